"""On-policy replicas on CPU (gloo, world size 2): rank 0's weights for all, one flattened all-reduce per optimiser step, advantages
normalised over all ranks, identical weights after training on different episodes, equal (to float32 rounding) to one process
trained on the episodes joined.  Plain torch forms stand in for the device operators."""
import math
import os
import sys
import types

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBS, HID, T, E, N, EPOCHS = 12, 8, 9, 3, 4, 3


def _gated_scan(gate, x, h0=None, *, resets=None):
    h, out = torch.zeros_like(x[0]), []
    for t in range(x.shape[0]):
        a = torch.sigmoid(gate[t])
        h = a * h + (1 - a) * x[t]
        out.append(h)
    return torch.stack(out), h


def _policy_loss(mean, log_std, actions, old, adv, *, adv_moments, clip, kl_coef, entropy_coef):
    z = (actions - mean) * torch.exp(-log_std)
    lp = (-z * z / 2 - log_std - math.log(2 * math.pi) / 2).sum(-1)
    A, q, D = (adv - adv_moments[0]) * adv_moments[1], torch.exp(lp - old), old - lp
    gain, k = torch.minimum(q * A, q.clamp(1 - clip, 1 + clip) * A).mean(), (torch.expm1(D) - D).mean()
    H = (log_std + (1 + math.log(2 * math.pi)) / 2).sum()
    return -gain + kl_coef * k - entropy_coef * H, torch.stack([gain, k, H, 0 * k, q.mean(), 0 * k]).detach()


def _episode(seed, envs=E):
    """What train_on_policy reads of an environment and a replay."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    obs, act, lp, rew = rn(T + 1, envs, OBS, N), rn(T, envs, 2, N), -2.5 + 0.1 * rn(T, envs, N), rn(T, envs, N) * (1 + seed)
    return obs, act, lp, rew


def _replay(obs, act, lp, rew):
    def advantages(values, gamma, lam):
        adv = torch.zeros_like(rew)
        run = torch.zeros_like(rew[0])
        for t in range(T - 1, -1, -1):
            run = rew[t] + gamma * values[t + 1] - values[t] + gamma * lam * run
            adv[t] = run
        return adv, adv + values[:-1], torch.stack([adv.double().mean(), 1 / (adv.double().std(unbiased=False) + 1e-8)]).float()
    env = types.SimpleNamespace(E=obs.shape[1], n_a=N, device="cpu")
    return env, types.SimpleNamespace(slot=0, complete=[True], T=T, obs_ring=obs.unsqueeze(0), act_ring=act.unsqueeze(0), log_pi_ring=lp.unsqueeze(0), advantages=advantages)


def _learner(**kw):
    sys.path.insert(0, REPO)
    from marl_amd import rollout
    rollout.gated_scan, rollout.clipped_policy_loss = _gated_scan, _policy_loss
    return rollout, rollout.ClippedPolicyLearner(OBS, hidden_dim=HID, kl_coef=0.1, entropy_coef=0.01, device="cpu", **kw)


def _weights(L):
    return torch.cat([p.detach().reshape(-1) for net in (L.policy, L.critic) for p in net.parameters()]).numpy()


def _worker(rank, world, port, out):
    os.environ["MASTER_ADDR"] = "127.0.0.1"; os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    torch.manual_seed(100 + rank)                                     # replicas start DIFFERENT until rank 0's weights arrive
    rollout, L = _learner(data_parallel=True)
    calls = []
    real = dist.all_reduce
    dist.all_reduce = lambda t, *a, **k: (calls.append(t.numel()), real(t, *a, **k))[1]
    rollout.train_on_policy(*_pair(L, rank), epochs=EPOCHS, envs_per_batch=E)
    dist.all_reduce = real
    sizes = [sum(p.numel() for p in net.parameters()) for net in (L.policy, L.critic)]
    refused = []
    env, replay = _replay(*_episode(rank, E + rank))                  # (a different number of environments on each rank)
    try:
        rollout.train_on_policy(env, L, replay, epochs=1, envs_per_batch=2)
    except RuntimeError as e:
        refused.append(str(e))
    _, alone = _learner()
    env, replay = _replay(*_episode(rank))
    try:
        rollout.train_on_policy(env, alone, replay, epochs=1)
    except RuntimeError as e:
        refused.append(str(e))
    same = rollout._over_ranks(torch.tensor([777.7, 1e8]), (1,), None)      # (equal everywhere: no deviation appears)
    assert same.tolist() == torch.tensor([777.7, 1e8]).tolist()
    two = rollout._over_ranks(torch.tensor([5.0 + rank, 1 / (2.0 + 1e-8)]), (1,), None)
    assert two.tolist() == pytest.approx([5.5, 1 / (4.25 ** 0.5 + 1e-8)], rel=1e-6)
    own = [dist.new_group([r]) for r in range(world)][rank]
    _, single = _learner(group=own)                                   # a group of this rank alone: nothing to drift from
    rollout.train_on_policy(env, single, replay, epochs=1)
    out.put((rank, _weights(L), calls == [10 + 2 * world] + sizes * EPOCHS, refused))
    dist.barrier()
    dist.destroy_process_group()


def _pair(L, rank):
    env, replay = _replay(*_episode(rank))
    return env, L, replay


def test_replicas_train_as_one():
    world = 2
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 35500 + os.getpid() % 2000
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = {r: rest for r, *rest in (q.get(timeout=180) for _ in range(world))}
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for r in range(world):
        assert got[r][1], "one message with the moments, then one flattened all-reduce per optimiser step"
        assert len(got[r][2]) == 2 and "differ" in got[r][2][0] and "data_parallel=True" in got[r][2][1], got[r][2]
    assert np.array_equal(got[0][0], got[1][0]), "replicas diverged"
    from marl_amd import rollout
    keep = rollout.gated_scan, rollout.clipped_policy_loss
    try:
        torch.manual_seed(100)
        _, L = _learner()
        env, replay = _replay(*[torch.cat(p, 1) for p in zip(_episode(0), _episode(1))])
        rollout.train_on_policy(env, L, replay, epochs=EPOCHS, envs_per_batch=2 * E)
    finally:
        rollout.gated_scan, rollout.clipped_policy_loss = keep
    # (Adam divides by the root of a gradient's square: a rounding of it moves a weight by a part of the step, 1e-3 at most)
    np.testing.assert_allclose(got[0][0], _weights(L), rtol=2e-5, atol=2e-6)


def test_data_parallel_needs_a_process_group():
    with pytest.raises(RuntimeError, match="init_process_group"):
        sys.path.insert(0, REPO)
        from marl_amd.rollout import ClippedPolicyLearner
        ClippedPolicyLearner(OBS, hidden_dim=HID, device="cpu", data_parallel=True)
