"""BatchedSequenceDQNAgent on an env that is reset, stepped or sorted between two calls of collect."""
import pytest
import torch

pytestmark = pytest.mark.gpu
N = 64


def _agent(dev, auto_steps=24, **spec):
    from gym_PVDER_amd.agents import BatchedSequenceDQNAgent
    from gym_PVDER_amd.vec_env import PVDERVec
    env = PVDERVec(N, device=dev, n_sim_time_steps_per_env_step=15, max_sim_time=auto_steps / 4, seed=1, auto_reset=True)
    return env, BatchedSequenceDQNAgent(env, seed=0, **dict(dict(window=20, burn_in=4, replay_steps=64, batch_size=16), **spec))


def _memory_is_the_networks(agent, first, last):
    """The memory after steps first .. last of the buffer is what the network makes of them as a window."""
    from gym_PVDER_amd.agents.sequence import tokens_of
    x = tokens_of(agent.buf_obs[first:last], agent.buf_before[first:last], agent.buf_reward[first:last], agent.buf_start[first:last]).transpose(0, 1)
    with torch.no_grad():
        _, state = agent.q_net(x, starts=agent.buf_start[first:last].t(), output_state=True)
    for a, b in zip(state, agent.state):
        assert torch.isfinite(b).all()
        assert float((a - b).norm()) <= 2.0 ** -15 * float(b.norm())             # (the sums of 30 tokens in two orders)


def test_a_reset_of_some_envs_between_two_collects(gpu_device):
    env, agent = _agent(gpu_device)
    agent.collect(10, epsilon=1.0)
    rewards, done = env.out[11].clone(), env.out[12].clone()
    assert not done.any()
    mask = torch.arange(N, device=gpu_device) % 3 == 0
    env.reset(mask)
    agent.collect(10, epsilon=1.0)
    assert torch.equal(agent.buf_start[10], mask) and not agent.buf_start[1:10].any() and not agent.buf_start[11:20].any()
    assert torch.isnan(agent.buf_reward[10]).eq(mask).all() and torch.equal(agent.buf_reward[10][~mask], rewards[~mask])
    assert not torch.isnan(agent.buf_reward[:10]).any() and not torch.isnan(agent.buf_reward[11:]).any()
    _memory_is_the_networks(agent, 0, 20)
    agent.collect(2)
    tokens, starts, actions, r = agent.sample()
    assert torch.isfinite(tokens).all() and torch.isfinite(agent.loss(tokens, starts, actions, r))
    agent.collect(2)                                                             # nothing happened in between: the episode of step 20 goes on
    assert not agent.buf_start[20:24].any()


def test_a_new_event_grid_between_two_collects(gpu_device):
    """The env resets at the next collect: the last actions before it have no known outcome, and are no ends of episodes."""
    env, agent = _agent(gpu_device)
    agent.collect(10, epsilon=1.0)
    env.update_env_events([{"voltage": {"t_events_step": 0.5}}])
    assert env._needs_reset
    agent.collect(10, epsilon=1.0)
    assert agent.buf_start[10].all() and torch.isnan(agent.buf_reward[10]).all()
    _memory_is_the_networks(agent, 0, 20)


def test_an_episode_that_ended_keeps_its_last_reward(gpu_device):
    env, agent = _agent(gpu_device)
    agent.collect(24, epsilon=1.0)
    assert env.out[12].all()                                                     # every env finished, and was reset in the same launch
    rewards = env.out[11].clone()
    env.reset()
    agent.collect(4, epsilon=1.0)
    assert agent.buf_start[24].all() and torch.equal(agent.buf_reward[24], rewards)


def test_new_events_in_a_running_episode_do_not_cut_it(gpu_device):
    env, agent = _agent(gpu_device)
    agent.collect(10, epsilon=1.0)
    rewards = env.out[11].clone()
    env.update_env_events([{"voltage": {"max": 1.03}}])
    assert not env._needs_reset
    agent.collect(4, epsilon=1.0)
    assert not agent.buf_start[1:14].any() and torch.equal(agent.buf_reward[10], rewards)


def test_steps_taken_elsewhere_and_another_output_block(gpu_device):
    env, agent = _agent(gpu_device)
    agent.collect(6, epsilon=1.0)
    obs = env.out[:11].clone()
    env.use_out(torch.full_like(env.out, 7.0))                                   # holds nothing of the env yet
    agent.collect(2, epsilon=1.0)
    assert not agent.buf_start[1:8].any() and torch.equal(agent.buf_obs[6], obs.t())
    env.step(torch.ones(N, dtype=torch.uint8, device=gpu_device))
    agent.collect(2, epsilon=1.0)
    assert agent.buf_start[8].all() and torch.isnan(agent.buf_reward[8]).all()


@pytest.mark.parametrize("lane_io", [False, True])
def test_sorted_lanes_change_no_evaluation(gpu_device, lane_io):
    from gym_PVDER_amd.vec_env import PVDERVec
    _, agent = _agent(gpu_device)
    returns = []
    for sort in (False, True):
        env = PVDERVec(N, device=gpu_device, n_sim_time_steps_per_env_step=15, max_sim_time=6.0, seed=5, auto_reset=False)
        env.reset()
        if sort:
            env.sort_lanes(key=torch.arange(N, 0, -1), lane_io=lane_io)
        returns.append(agent.evaluate(env)["returns"])
    assert torch.equal(*returns) and len(set(returns[0].tolist())) > 1


@pytest.mark.parametrize("lane_io", [False, True])
def test_sorted_lanes_change_nothing(gpu_device, lane_io):
    agents = []
    for sort in (False, True):
        env, agent = _agent(gpu_device)
        agent.collect(5, epsilon=0.5)
        env.reset(torch.arange(N, device=gpu_device) % 5 == 2)
        agent.collect(5, epsilon=0.5)
        if sort:
            env.sort_lanes(lane_io=lane_io)
            assert not torch.equal(env.env_of_lane.long(), torch.arange(N, device=gpu_device))
        agent.collect(25, epsilon=0.5)                                           # past ends of episodes
        agents.append(agent)
    a, b = agents
    for n in ("buf_obs", "buf_before", "buf_action", "buf_start"):
        assert torch.equal(getattr(a, n), getattr(b, n)), n
    assert torch.equal(torch.nan_to_num(a.buf_reward, 5.0), torch.nan_to_num(b.buf_reward, 5.0))
    assert all(torch.equal(x, y) for x, y in zip(a.state, b.state))


def test_the_loss_leaves_out_what_is_not_known(gpu_device):
    env, agent = _agent(gpu_device, gamma=0.9)
    agent.collect(12, epsilon=1.0)
    env.reset()
    agent.collect(30, epsilon=1.0)
    tokens, starts, actions, rewards = agent.sample()
    cut = torch.isnan(rewards)
    assert cut.any() and not cut.all() and not (cut & ~starts[:, 1:]).any()
    loss = agent.loss(tokens, starts, actions, rewards)
    grads = torch.autograd.grad(loss, list(agent.q_net.parameters()))
    assert all(torch.isfinite(g).all() for g in grads)
    with torch.no_grad():
        after = agent.target(tokens, starts=starts).double()[:, 1:].amax(2).masked_fill(starts[:, 1:], 0.0)
        values = agent.q_net(tokens[:, :-1], starts=starts[:, :-1]).double().gather(2, actions[:, :-1, None].long())[..., 0]
        off = (values - rewards.double() - 0.9 * after)[:, 4:][~cut[:, 4:]]
        # float32 differences of numbers below their magnitudes' sum, squared: 6 roundings of each term's size
        size = ((values.abs() + rewards.double().abs() + after.abs())[:, 4:][~cut[:, 4:]] ** 2).mean()
        assert abs(float(loss) - float((off ** 2).mean())) <= 16 * 2.0 ** -24 * float(size) + 1e-12
    nothing = agent.loss(tokens, starts, actions, torch.full_like(rewards, float("nan")))
    assert float(nothing.detach()) == 0.0


def test_an_env_of_64_bits(gpu_device):
    from gym_PVDER_amd.agents import BatchedSequenceDQNAgent
    from gym_PVDER_amd.vec_env import PVDERVec
    env = PVDERVec(8, device=gpu_device, integrator="etdlin64", n_sim_time_steps_per_env_step=15, max_sim_time=6.0, seed=1, auto_reset=True)
    agent = BatchedSequenceDQNAgent(env, seed=0, window=6, burn_in=2, replay_steps=16, batch_size=4)
    agent.collect(4, epsilon=1.0)
    mask = torch.arange(8, device=gpu_device) < 3
    env.reset(mask)
    agent.collect(4, epsilon=1.0)
    assert torch.equal(agent.buf_start[4], mask) and torch.equal(torch.isnan(agent.buf_reward[4]), mask) and not agent.buf_start[5:8].any()
    assert torch.isfinite(torch.tensor(agent.train_step()))
