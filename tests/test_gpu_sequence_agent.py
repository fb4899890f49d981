"""The agent with a memory: its network as a run of the sequence operators together, and its loop."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _plain(net, tokens, starts, lengths=None, state=None):
    """SequenceQNetwork.forward written out in 64 bits with torch's own operations (differentiable): (values, states)."""
    p = {n: x.detach().double().cpu().requires_grad_() for n, x in net.named_parameters()}
    rms = lambda z, w: z * ((z * z).mean(-1, keepdim=True) + 1e-6) ** -0.5 * w  # noqa: E731
    x = tokens.double().cpu()
    B, T = x.shape[:2]
    g = net.log_decay.double().cpu().exp().view(1, -1, 1, 1)
    lengths = torch.full((B,), T) if lengths is None else lengths.cpu()
    h = F.linear(x, p["embed"], p["embed_bias"])
    u = rms(h, p["pre"])
    inner, states = net.heads * net.head_dim, []
    for i in range(len(net.blocks)):
        b = {n: p["blocks.%d.%s" % (i, n)] for n in ("project", "out", "post", "pre", "scale")}
        w = F.linear(u, b["project"])
        q, k, v = (w[..., j * inner:(j + 1) * inner].unflatten(-1, (net.heads, net.head_dim)) for j in range(3))
        S = torch.zeros(B, net.heads, net.head_dim, net.head_dim, dtype=torch.float64) if state is None else state[i].double().cpu()
        o = []
        for t in range(T):
            keep, on = (~starts[:, t].cpu()).double().view(B, 1, 1, 1), (t < lengths).double().view(B, 1, 1, 1)
            S = on * (keep * g * S + k[:, t, :, :, None] * v[:, t, :, None, :]) + (1 - on) * S
            o.append(on[..., 0] * torch.einsum("bhi,bhij->bhj", q[:, t], S) * net.head_dim ** -0.5)
        states.append(S)
        y = F.linear(torch.stack(o, 1).flatten(-2), b["out"])
        h = h + b["scale"] * torch.sigmoid(w[..., 3 * inner:]) * rms(y, b["post"])
        u = rms(h, b["pre"])
    return F.linear(u, p["head"], p["head_bias"]), states, p


def _windows(B, T, dev, seed=0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    starts = torch.rand(B, T, generator=g) < 0.05
    return torch.randn(B, T, 17, generator=g).to(dev), starts.to(dev)


# A value passes 2 blocks of 7 operations (projection, attention, product, two norms, gate, sum) and 3 more outside: 17 results, each
# off by a few roundings of its terms (sums of at most 130 of them, of both signs).  Relative to the norm of the whole, 17 times 8
# roundings is generous to every one of them: 17 * 8 * 2^-24 = 8e-6; with bf16 in the blocks 17 roundings of 2^-8 = 0.066.
TOL = {torch.float32: 17 * 8 * 2.0 ** -24, torch.bfloat16: 17 * 2.0 ** -8}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,heads,head_dim", [(64, 4, 16), (100, 3, 20)])
def test_network_and_its_gradients(gpu_device, width, heads, head_dim, dtype):
    from gym_PVDER_amd.agents import SequenceQNetwork
    net = SequenceQNetwork(width, heads, head_dim, compute_dtype=dtype, device=gpu_device, seed=3)
    x, starts = _windows(5, 70, gpu_device)
    lengths = torch.tensor([70, 64, 1, 33, 70], dtype=torch.int32, device=gpu_device)
    values, states = net(x, starts=starts, lengths=lengths, output_state=True)
    want, ws, p = _plain(net, x, starts, lengths)
    rel = lambda a, b: float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert rel(values, want) < TOL[dtype]
    for a, b in zip(states, ws):
        assert rel(a, b) < TOL[dtype]
    weight = torch.randn(values.shape, generator=torch.Generator().manual_seed(1))
    values.backward(weight.to(gpu_device))
    want.backward(weight.double())
    for n, q in net.named_parameters():
        assert rel(q.grad, p[n].grad) < 2 * TOL[dtype], n                # forward and backward


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_are_the_window(gpu_device, dtype):
    """Acting step by step sees what training on the window sees, from a memory that another window left."""
    from gym_PVDER_amd.agents import SequenceQNetwork
    net = SequenceQNetwork(compute_dtype=dtype, device=gpu_device)
    x, starts = _windows(6, 90, gpu_device, 4)
    with torch.no_grad():
        whole = net(x, starts=starts)
        _, state = net(x[:, :50], starts=starts[:, :50], output_state=True)
    got = torch.stack([net.step(x[:, t], state, starts[:, t]) for t in range(50, 90)], 1)
    assert float((got - whole[:, 50:]).norm() / whole[:, 50:].norm()) < 2 * TOL[dtype]


def test_a_captured_training_step(gpu_device):
    """Forward and backward of the network in a graph, replayed with new windows between eager passes of other leaves."""
    from gym_PVDER_amd.agents import SequenceQNetwork
    net, other = (SequenceQNetwork(device=gpu_device, seed=s) for s in (1, 2))
    x, starts = _windows(8, 60, gpu_device)
    params = list(net.parameters())

    def grads(n):
        return torch.autograd.grad(n(x, starts=starts).square().mean(), list(n.parameters()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(net)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = torch.autograd.grad(net(x, starts=starts).square().mean(), params)
    for turn in range(3):
        x.copy_(_windows(8, 60, gpu_device, 10 + turn)[0])
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        grads(other)
        for a, b in zip(got, grads(net)):
            assert float((a - b).norm()) <= 1e-5 * float(b.norm()) + 1e-12
        torch.cuda.synchronize()


def test_agent_collects_trains_and_evaluates(gpu_device):
    from gym_PVDER_amd.agents import BatchedSequenceDQNAgent
    from gym_PVDER_amd.agents.sequence import tokens_of
    from gym_PVDER_amd.vec_env import PVDERVec
    env = PVDERVec(64, device=gpu_device, n_sim_time_steps_per_env_step=15, max_sim_time=6.0, seed=1, auto_reset=True)
    agent = BatchedSequenceDQNAgent(env, seed=0, window=20, burn_in=4, replay_steps=48, batch_size=16)
    agent.collect(48 + 13, epsilon=1.0)                                  # past the ring's end
    assert agent.steps_in == 48 and agent.at == 13
    # the ring in order: an env's token holds the action stored with the token before, and an episode is 24 steps
    order = (torch.arange(48, device=gpu_device) + 13) % 48
    assert torch.equal(agent.buf_before[order][1:], agent.buf_action[order][:-1])
    assert int(agent.buf_start.sum()) in (2 * 64, 2 * 64 + 64)
    tokens, starts, actions, rewards = agent.sample()
    assert tokens.shape == (16, 21, 17) and rewards.shape == (16, 20)
    assert not tokens[..., 11:][starts].any() and torch.equal(tokens[:, 1:, 16][~starts[:, 1:]], rewards[~starts[:, 1:]])
    # the memory that acting has built is that of the network over the running episodes
    at = order[-24:]
    x = tokens_of(agent.buf_obs[at], agent.buf_before[at], agent.buf_reward[at], agent.buf_start[at]).transpose(0, 1)
    with torch.no_grad():
        _, state = agent.q_net(x, starts=agent.buf_start[at].t(), output_state=True)
    for a, b in zip(state, agent.state):
        assert float((a - b).norm() / b.norm()) < 2 * TOL[torch.float32]
    before = [p.detach().clone() for p in agent.q_net.parameters()]
    losses = agent.train(3, initial_collect_steps=1)
    assert len(losses) == 3 and all(torch.isfinite(torch.tensor(losses)))
    assert all(not torch.equal(a, b) for a, b in zip(before, agent.q_net.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(agent.target.parameters(), agent.q_net.parameters()))
    r = agent.evaluate(PVDERVec(32, device=gpu_device, n_sim_time_steps_per_env_step=15, max_sim_time=6.0, seed=5, auto_reset=False))
    assert r["returns"].shape == (32,) and r["min"] <= r["average_return"] <= r["max"]


def test_agent_refuses(gpu_device):
    from gym_PVDER_amd.agents import BatchedSequenceDQNAgent, SequenceQNetwork
    from gym_PVDER_amd.vec_env import PVDERVec
    env = PVDERVec(4, device=gpu_device, auto_reset=True)
    for bad in (dict(window=16, burn_in=16), dict(window=512), dict(no_such=1), dict(head_dim=129), dict(compute_dtype=torch.float16)):
        with pytest.raises(ValueError):
            BatchedSequenceDQNAgent(env, **bad)
    with pytest.raises(TypeError):
        BatchedSequenceDQNAgent(None)
    with pytest.raises(ValueError):
        SequenceQNetwork(horizons=(1.0, 5.0), device=gpu_device)
    with pytest.raises(ValueError, match="collect more"):
        BatchedSequenceDQNAgent(env).sample()
