"""The limits of the sequence operators' C entries against each other.  Runs on the CPU: every call here is refused, at the
latest for its NULL pointers, before anything is launched."""
from marl_amd import _lib


def test_what_the_loss_takes_its_scaling_takes():
    """2^29 rows of up to 32 components: the gradients to scale are 32 x 2^29 values."""
    lib = _lib.load()
    for rows, A in ((1 << 29, 1), ((1 << 28) + 1, 2), ((1 << 24) + 1, 32), (1 << 29, 32)):
        assert lib.asm_policy_loss_workspace(rows, A) > 0
        for n_std in (A, rows * A):
            for dtype in (_lib.SEQ_F32, _lib.SEQ_BF16):
                assert lib.asm_policy_loss_scale(dtype, None, rows * A, None, n_std, None, None) != 0
                assert "too large" not in lib.asm_last_error().decode(), (rows, A, n_std)
    for n_mean, n_std in ((-1, 2), (2, -1), ((32 << 29) + 1, 2), (2, (32 << 29) + 1)):
        assert lib.asm_policy_loss_scale(_lib.SEQ_F32, None, n_mean, None, n_std, None, None) != 0
        assert "too large" in lib.asm_last_error().decode()
    assert lib.asm_policy_loss_scale(7, None, 2, None, 2, None, None) != 0 and "dtype" in lib.asm_last_error().decode()
