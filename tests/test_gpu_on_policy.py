"""The sequence operators together, as a program uses them: an episode run under a policy with a memory (gated_scan_step,
gaussian_act), recorded in the replay, its advantages, the clipped loss over the whole episode and its gradients
(gated_scan, clipped_policy_loss), against the same computation in 64 bits on the CPU."""
import math

import pytest

import seq_oracle as so

pytestmark = pytest.mark.gpu
T, E, N, H = 20, 6, 30, 64


def _setup(torch, E=E, episodes=1, sharded=False):
    from marl_amd.batched import BatchedAssemblyEnv
    from marl_amd.replay import DeviceReplay
    from marl_amd.rollout import ClippedPolicyLearner, run_episode
    from marl_amd.sharding import StreamShards
    torch.manual_seed(7)
    env = StreamShards(E, N, parts=2, seed=3) if sharded else BatchedAssemblyEnv(E, N, seed=3)
    dim = env.envs[0].obs_dim_agent if sharded else env.obs_dim_agent
    learner = ClippedPolicyLearner(dim, hidden_dim=H, kl_coef=0.1, entropy_coef=0.01)
    replay = DeviceReplay(env, T, 2, log_pi=True)
    for _ in range(episodes):
        stats = run_episode(env, learner, replay, T)
    assert bool(torch.isfinite(torch.as_tensor(stats)).all())
    return env, learner, replay


def _policy64(torch, policy, rows):
    """MemoryPolicy.forward in float64 on the CPU, with gradients."""
    import torch.nn.functional as F
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in policy.named_parameters()}
    x = rows.detach().cpu().double()
    z = F.leaky_relu(x @ p["fc1.weight"].t() + p["fc1.bias"]) @ p["fc2.weight"].t() + p["fc2.bias"]
    g, u = z.chunk(2, -1)
    a = torch.sigmoid(g)
    h, hs = torch.zeros_like(u[0]), []
    for t in range(x.shape[0]):
        h = a[t] * h + (1 - a[t]) * u[t]
        hs.append(h)
    return torch.tanh(torch.stack(hs) @ p["fc4.weight"].t() + p["fc4.bias"]), p


def test_an_episode_and_its_gradients(torch_cuda):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    env, learner, replay = _setup(torch)
    frames, acts, lp = replay.obs_ring[0], replay.act_ring[0], replay.log_pi_ring[0]
    rows = learner._rows(frames[:T])
    mean, last = learner.policy(rows)
    mean64, p = _policy64(torch, learner.policy, rows)
    # products of 192 and 64 terms of order 1 and a memory that averages: errors of a few times sqrt(192) u, held to 100 u
    assert float((mean.detach().cpu().double() - mean64.detach()).abs().max()) < 100 * so.U * 4
    # the rollout's memory, step by step, is the sequence's
    assert float((learner._states[0] - last).detach().abs().max()) < 100 * so.U * float(last.detach().abs().max() + 1)
    # the recorded log_pi is that of the recorded actions under the mean of the step-by-step policy: a mean off by e moves it by |z| e / std
    want = so.log_pi(mean64.view(T, E, N, 2), learner.policy.log_std, acts.transpose(-1, -2))
    z = (acts.transpose(-1, -2).cpu().double() - mean64.view(T, E, N, 2)).abs().sum(-1) / 0.25
    assert bool(((lp.cpu().double() - want).abs() <= 400 * so.U * (z + 1) + so.U * want.abs()).all())
    # advantages from the replay
    values = torch.randn(T + 1, E, N, device="cuda")
    adv, ret, mom = replay.advantages(values)
    wa, ta, wr, tr, _, _ = so.advantages(replay.rew_ring[0].squeeze(2), values)
    so.within(adv, wa, ta, "adv"); so.within(ret, wr, tr, "ret")
    # at the first update the ratio is 1 and the KL estimate 0
    loss, stats = clipped_policy_loss(mean.view(T, E, N, 2), learner.policy.log_std, acts.transpose(-1, -2), lp, adv, adv_moments=mom, kl_coef=0.1, entropy_coef=0.01)
    st = dict(zip(("gain", "kl", "entropy", "clipped", "ratio", "rows"), stats.tolist()))
    assert abs(st["ratio"] - 1.0) < 1e-4 and 0 <= st["kl"] < 1e-8 and st["clipped"] == 0 and st["rows"] == T * E * N
    # a policy some updates on: gradients of every parameter through loss and memory
    with torch.no_grad():
        old = lp + 0.2 * torch.randn_like(lp)
    loss, _ = clipped_policy_loss(mean.view(T, E, N, 2), learner.policy.log_std, acts.transpose(-1, -2), old, adv, adv_moments=mom, kl_coef=0.1, entropy_coef=0.01)
    grads = torch.autograd.grad(loss, list(learner.policy.parameters()))
    m, s = mean64.view(T, E, N, 2), p["log_std"]
    a64 = acts.transpose(-1, -2).cpu().double()
    l64 = (-((a64 - m) / s.exp()) ** 2 / 2 - s - math.log(2 * math.pi) / 2).sum(-1)
    A = (adv.cpu().double() - mom[0].cpu().double()) * mom[1].cpu().double()
    D = old.cpu().double() - l64
    q = torch.exp(-D)
    want = (-torch.minimum(q * A, q.clamp(0.8, 1.2) * A) + 0.1 * (torch.expm1(D) - D)).mean() - 0.01 * (s + (1 + math.log(2 * math.pi)) / 2).sum()
    g64 = torch.autograd.grad(want, list(p.values()))
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    for (name, _), a, b in zip(learner.policy.named_parameters(), grads, g64):
        # float32 products over 3600 rows; rows whose float32 mean puts them on the other side of the clipping border: at most 1e-5 of them
        off = float((a.detach().cpu().double() - b).norm() / b.norm().clamp_min(1e-12))
        assert off < 1e-3, (name, off)


@pytest.mark.parametrize("sharded", [False, True])
def test_training_runs(torch_cuda, sharded):
    torch = torch_cuda
    from marl_amd.rollout import eval_episode, run_episode, train_on_policy
    env, learner, replay = _setup(torch, 8, 2, sharded)
    before = [p.detach().clone() for p in learner.policy.parameters()]
    for epoch in range(2):
        run_episode(env, learner, replay, T)
        losses = train_on_policy(env, learner, replay, epochs=2, envs_per_batch=3)
        assert losses.shape == (6, 8) and bool(torch.isfinite(losses).all())
        assert abs(float(losses[0, 6]) - 1.0) < 1e-4                   # the first update of an episode starts at ratio 1
    assert all(not torch.equal(a, b) for a, b in zip(before, learner.policy.parameters()))
    if not sharded:
        metrics, total = eval_episode(env, learner, 5)
        assert metrics.shape == (5, 8, 5) and bool(torch.isfinite(total).all())
        a, b = (torch.empty(8, 2, N, device="cuda") for _ in range(2))
        learner.begin_episode(); learner.act(env.reset(0), a)
        learner.begin_episode(); learner.act(env.reset(0), b)
        assert torch.equal(a, b)                                        # the memory starts empty each time


def test_sharded_episode_is_the_unsharded_one(torch_cuda):
    """Shards of one size step and act at the same time, each with its own memory and its own rows: without noise the episode
    is the one of a single environment of all."""
    torch = torch_cuda
    out = []
    for sharded in (False, True):
        env, learner, replay = _setup(torch, 64, 1, sharded)
        envs = env.envs if sharded else [env]
        learner.begin_episode()
        a = torch.empty(64, 2, N, device="cuda")
        obs = list(env.reset(5)) if sharded else [env.reset(5)]
        torch.cuda.synchronize()
        frames = []
        for t in range(6):
            first = 0
            for k, e in enumerate(envs):
                ak = a[first:first + e.E]
                st = env.streams[k] if sharded else torch.cuda.current_stream()
                with torch.cuda.stream(st):
                    learner.act(obs[k], ak, env0=e.env_id_offset)
                    obs[k] = e.step(ak)[0].clone()
                first += e.E
            torch.cuda.synchronize()
            frames.append(a.clone())
        out.append(torch.stack(frames))
    # (a matrix product over half the rows may sum in another order: 64-term sums of order 1)
    assert float((out[0] - out[1]).abs().max()) < 100 * so.U * 4


def test_what_is_refused(torch_cuda):
    torch = torch_cuda
    from marl_amd.batched import BatchedAssemblyEnv
    from marl_amd.replay import DeviceReplay
    from marl_amd.rollout import ClippedPolicyLearner, run_episode, train_on_policy
    env = BatchedAssemblyEnv(2, N, seed=1)
    learner = ClippedPolicyLearner(env.obs_dim_agent, hidden_dim=H)
    plain, replay = DeviceReplay(env, 3, 1), DeviceReplay(env, 3, 1, log_pi=True)
    with pytest.raises(RuntimeError, match="log_pi"):
        run_episode(env, learner, plain, 3)
    with pytest.raises(ValueError, match="noise_scale"):
        run_episode(env, learner, replay, 3, noise_scale=0.0)
    with pytest.raises(RuntimeError, match="complete episode"):
        train_on_policy(env, learner, replay)
    with pytest.raises(RuntimeError, match="complete episode"):
        replay.advantages(torch.zeros(4, 2, N, device="cuda"))
