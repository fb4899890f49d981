"""A DQN agent with a memory, over a PVDERVec: the loop of :class:`~gym_PVDER_amd.agents.dqn.BatchedDQNAgent` (the reference's
TF-Agents demo, /root/reference/examples/gym_PVDER_environment_tf_agents_DQN_demo.ipynb cells 12-28) with a network that sees the
whole episode so far instead of one observation.

An observation does not show what an env with randomised parameters is made of, nor where the grid has been going; the steps of the
running episode do.  :class:`SequenceQNetwork` reads a token per env step -- the observation, the action that led to it and its reward
-- and answers with the five action values.  Its blocks are a decay attention (``sequence_ops.decay_attention``: the memory of an env
has a fixed size) and the residual stream between them (``sequence_ops.gated_residual_norm``):

    u = rms(embed(token)),  h = embed(token)
    q, k, v, gate = project(u);  y = out(decay_attention(q, k, v));  h, u = gated_residual_norm(h, y, gate)      for each block
    action values = head(u)

* acting: :meth:`SequenceQNetwork.step`, one token of every env, the memory updated in place (65 536 envs, four heads of 32 x 32:
  one GB of memory read and written per block);
* training: :meth:`SequenceQNetwork.forward` on windows of the replay buffer, all tokens at once, episodes that end and start inside
  kept apart by ``starts``.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch
import torch.nn.functional as F

from ..vec_env import PVDERVec
from .dqn import N_ACT, N_OBS
from .sequence_ops import decay_attention, decay_attention_step, gated_residual_norm

N_TOKEN = N_OBS + N_ACT + 1                # observation, one-hot of the action before, its reward
EPS = 1e-6


def tokens_of(obs: torch.Tensor, action: torch.Tensor, reward: torch.Tensor, starts: torch.Tensor) -> torch.Tensor:
    """Observations [..., 11], the actions and rewards before them [...] and where episodes start [...] -> tokens [..., 17]; the first
    token of an episode has no action and no reward before it."""
    before = torch.cat([F.one_hot(action.long(), N_ACT).to(obs.dtype), reward.to(obs.dtype)[..., None]], -1)
    return torch.cat([obs, before.masked_fill(starts.bool()[..., None], 0.0)], -1)


class SequenceBlock(torch.nn.Module):
    def __init__(self, width: int, heads: int, head_dim: int):
        super().__init__()
        inner = heads * head_dim
        self.project = torch.nn.Parameter(torch.empty(3 * inner + width, width))        # q, k, v, gate
        self.out = torch.nn.Parameter(torch.empty(width, inner))
        self.post = torch.nn.Parameter(torch.ones(width))
        self.pre = torch.nn.Parameter(torch.ones(width))
        self.scale = torch.nn.Parameter(torch.full((width,), 0.5))


class SequenceQNetwork(torch.nn.Module):
    """Tokens [..., 17] -> action values [..., 5].  ``compute_dtype`` bfloat16 runs the blocks in bf16 on fp32 weights; the memory is
    fp32 either way.  ``horizons``: over how many env steps the first and the last head forget (1 / (1 - decay))."""

    def __init__(self, width: int = 64, heads: int = 4, head_dim: int = 16, blocks: int = 2, horizons: Sequence[float] = (4.0, 128.0),
                 compute_dtype: torch.dtype = torch.float32, device="cuda", seed: int = 0):
        super().__init__()
        if compute_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("compute_dtype must be float32 or bfloat16")
        if min(width, heads, head_dim, blocks) < 1 or head_dim > 128 or width > 8192:
            raise ValueError("width must be in 1..8192, head_dim in 1..128, heads and blocks at least 1")
        if len(horizons) != 2 or not all(1.0 < x < float("inf") for x in horizons):
            raise ValueError("horizons are two finite numbers of env steps above 1")
        self.width, self.heads, self.head_dim, self.compute_dtype = int(width), int(heads), int(head_dim), compute_dtype
        self.embed = torch.nn.Parameter(torch.empty(width, N_TOKEN))
        self.embed_bias = torch.nn.Parameter(torch.zeros(width))
        self.pre = torch.nn.Parameter(torch.ones(width))
        self.blocks = torch.nn.ModuleList([SequenceBlock(width, heads, head_dim) for _ in range(blocks)])
        self.head = torch.nn.Parameter(torch.empty(N_ACT, width))
        self.head_bias = torch.nn.Parameter(torch.full((N_ACT,), -0.2))
        self.register_buffer("log_decay", torch.log1p(-1.0 / torch.logspace(*torch.log10(torch.tensor(horizons, dtype=torch.float64)).tolist(), heads,
                                                                               dtype=torch.float64)).to(torch.float32))
        g = torch.Generator(device="cpu")
        g.manual_seed(seed)
        with torch.no_grad():
            for name, p in self.named_parameters():
                if p.dim() == 2:
                    bound = 0.03 if name == "head" else (3.0 / p.shape[1]) ** 0.5        # (the demo's output layer: uniform in +-0.03)
                    p.copy_((torch.rand(p.shape, generator=g) * 2 - 1) * bound)
        self.to(device)

    def init_state(self, num_envs: int) -> List[torch.Tensor]:
        """An empty memory of every env, one tensor for each block."""
        return [torch.zeros((num_envs, self.heads, self.head_dim, self.head_dim), dtype=torch.float32, device=self.embed.device) for _ in self.blocks]

    def _run(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        dt = self.compute_dtype
        h = F.linear(tokens.to(dt), self.embed.to(dt), self.embed_bias.to(dt))
        u = F.rms_norm(h.float(), (self.width,), self.pre, EPS).to(dt)
        inner = self.heads * self.head_dim
        for i, b in enumerate(self.blocks):
            p = F.linear(u, b.project.to(dt))
            q, k, v = (p[..., j * inner:(j + 1) * inner].unflatten(-1, (self.heads, self.head_dim)) for j in range(3))
            y = F.linear(attend(i, q, k, v).flatten(-2), b.out.to(dt))
            h, u = gated_residual_norm(h, y, b.post, b.pre, gate=p[..., 3 * inner:], scale=b.scale, eps=EPS)
        return F.linear(u.float(), self.head, self.head_bias)

    def forward(self, tokens: torch.Tensor, state: Optional[List[torch.Tensor]] = None, starts: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, output_state: bool = False):
        """Windows [B, T, 17] -> action values [B, T, 5] (and the memory behind each window).  ``state``: the memory before it; ``starts``
        [B, T]: an episode starts here; ``lengths`` [B] int32: tokens of each window."""
        out_state: List[torch.Tensor] = []

        def attend(i, q, k, v):
            r = decay_attention(q, k, v, self.log_decay, initial_state=None if state is None else state[i], starts=starts, lengths=lengths,
                                output_final_state=output_state)
            if output_state:
                out_state.append(r[1])
                return r[0]
            return r

        values = self._run(tokens, attend)
        return (values, out_state) if output_state else values

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, state: List[torch.Tensor], starts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token of every env [N, 17] -> action values [N, 5]; ``state`` is updated in place, from nothing where ``starts``."""
        return self._run(tokens, lambda i, q, k, v: decay_attention_step(q, k, v, self.log_decay, state[i], starts=starts))


class BatchedSequenceDQNAgent:
    """DQN on :class:`SequenceQNetwork`.  The replay buffer holds whole batched steps, so that a window of any env can be read back;
    the first ``burn_in`` tokens of a window only fill the memory and are left out of the loss.

    The env may be reset, stepped, sorted (``sort_lanes``) or given other events between two calls of :meth:`collect`.  An env that is no
    longer where the last call left it starts an episode, and what its last action there would have led to is not known: the reward is
    stored as NaN, and :meth:`loss` leaves that action out.  Buffers and memory are in the order of the env ids."""

    train_spec = {'learning_rate': 1e-3, 'batch_size': 64, 'window': 160, 'burn_in': 16, 'replay_steps': 512, 'gamma': 1.0, 'epsilon_greedy': 0.1,
                  'target_update_period': 1, 'width': 64, 'heads': 4, 'head_dim': 16, 'blocks': 2, 'compute_dtype': torch.float32}

    def __init__(self, env: PVDERVec, seed: int = 0, **spec):
        if not isinstance(env, PVDERVec):
            raise TypeError("env must be a PVDERVec")
        unknown = set(spec) - set(self.train_spec)
        if unknown:
            raise ValueError("unknown settings: %s" % sorted(unknown))
        self.env, self.spec = env, dict(self.train_spec, **spec)
        sp, dev, N = self.spec, env.device, env.num_envs
        if not 0 <= sp['burn_in'] < sp['window'] < sp['replay_steps']:
            raise ValueError("0 <= burn_in < window < replay_steps must hold")
        net = lambda: SequenceQNetwork(sp['width'], sp['heads'], sp['head_dim'], sp['blocks'], compute_dtype=sp['compute_dtype'], device=dev, seed=seed)  # noqa: E731
        self.q_net, self.target = net(), net()
        self.optimizer = torch.optim.Adam(self.q_net.parameters(), lr=sp['learning_rate'])
        S = int(sp['replay_steps'])
        # step s of the ring: the token's observation, action before, reward before, start flag, and the action taken on it
        self.buf_obs = torch.zeros((S, N, N_OBS), dtype=torch.float32, device=dev)
        self.buf_before = torch.zeros((S, N), dtype=torch.uint8, device=dev)
        self.buf_reward = torch.zeros((S, N), dtype=torch.float32, device=dev)
        self.buf_start = torch.zeros((S, N), dtype=torch.bool, device=dev)
        self.buf_action = torch.zeros((S, N), dtype=torch.uint8, device=dev)
        self.steps_in, self.at = 0, 0                       # steps that the ring holds, and the next one's place
        self.state = self.q_net.init_state(N)
        self.action = torch.zeros(N, dtype=torch.uint8, device=dev)
        # of the next token: the reward behind that action, and whether an episode starts with it
        self.reward, self.start = torch.zeros(N, dtype=torch.float32, device=dev), torch.ones(N, dtype=torch.bool, device=dev)
        self.left = None                                    # where collect left the envs: output block, state, clock
        self.train_step_counter = 0
        self.gen = torch.Generator(device=dev)
        self.gen.manual_seed(seed + 1)

    def _act(self, values: torch.Tensor, epsilon: float) -> torch.Tensor:
        greedy = values.argmax(dim=1)
        if epsilon <= 0.0:
            return greedy.to(torch.uint8)
        n, dev = values.shape[0], values.device
        explore = torch.rand(n, generator=self.gen, device=dev) < epsilon
        return torch.where(explore, torch.randint(0, N_ACT, (n,), generator=self.gen, device=dev), greedy).to(torch.uint8)

    def collect(self, num_steps: int, epsilon: Optional[float] = None):
        """``num_steps`` batched env steps under the collect policy into the replay buffer."""
        env = self.env
        assert env.auto_reset, "construct the PVDERVec with auto_reset=True: collection runs across episode ends"
        eps = self.spec['epsilon_greedy'] if epsilon is None else epsilon
        if env._needs_reset:
            env.reset()
        out, state, clock = (env.to_env_order(t) for t in (env.out, env.fstate, env.istate[0]))
        if self.left is None:
            self.left = out.clone(), state.clone(), clock.clone()
            self.start.fill_(True)
        else:
            bits = torch.int64 if state.dtype == torch.float64 else torch.int32
            moved = (state.view(bits) != self.left[1].view(bits)).any(0) | (clock != self.left[2])
            self.reward.masked_fill_(moved & ~self.start, float("nan"))     # (an episode that had ended has its last reward)
            self.start |= moved
            out = torch.where(moved, out, self.left[0])     # (a block that ``use_out`` has put there holds no observation yet)
        for _ in range(num_steps):
            s = self.at
            self.buf_obs[s].copy_(out[:N_OBS].t())
            self.buf_before[s].copy_(self.action)
            self.buf_reward[s].copy_(self.reward)
            self.buf_start[s].copy_(self.start)
            tokens = tokens_of(self.buf_obs[s], self.buf_before[s], self.buf_reward[s], self.buf_start[s])
            self.action.copy_(self._act(self.q_net.step(tokens, self.state, self.buf_start[s]), eps))
            self.buf_action[s].copy_(self.action)
            env.step(env.to_lane_order(self.action) if env.lane_io else self.action, return_tensors=False)
            # (an env that finished has been reset in the same launch: its observation is the first of the next episode)
            out = env.to_env_order(env.out)
            self.reward.copy_(out[11])
            self.start.copy_(out[12] != 0)
            self.at = (s + 1) % self.buf_obs.shape[0]
            self.steps_in = min(self.steps_in + 1, self.buf_obs.shape[0])
        for mine, its in zip(self.left, (out, env.to_env_order(env.fstate), env.to_env_order(env.istate[0]))):
            mine.copy_(its)

    def sample(self):
        """``batch_size`` windows of ``window`` + 1 tokens: (tokens, starts, actions, rewards behind the actions, NaN where not known)."""
        sp, dev = self.spec, self.env.device
        B, T, S = int(sp['batch_size']), int(sp['window']) + 1, self.buf_obs.shape[0]
        if self.steps_in < T:
            raise ValueError("the buffer holds %d steps, a window needs %d: collect more" % (self.steps_in, T))
        first = torch.randint(0, self.steps_in - T + 1, (B, 1), generator=self.gen, device=dev)
        env = torch.randint(0, self.env.num_envs, (B, 1), generator=self.gen, device=dev)
        at = (self.at - self.steps_in + first + torch.arange(T, device=dev)) % S
        starts, reward = self.buf_start[at, env], self.buf_reward[at, env]
        tokens = tokens_of(self.buf_obs[at, env], self.buf_before[at, env], reward, starts)
        return tokens, starts, self.buf_action[at, env], reward[:, 1:]

    def loss(self, tokens, starts, actions, rewards) -> torch.Tensor:
        """Mean squared one-step error of the action values over the tokens behind ``burn_in``; the value of an episode's end is its
        reward, and an action whose reward is NaN does not count."""
        sp = self.spec
        with torch.no_grad():
            after = self.target(tokens, starts=starts)[:, 1:].max(dim=2).values
            wanted = rewards + sp['gamma'] * torch.where(starts[:, 1:], torch.zeros_like(after), after)
            known = ~torch.isnan(rewards)
        values = self.q_net(tokens[:, :-1], starts=starts[:, :-1]).gather(2, actions[:, :-1, None].long())[..., 0]
        off = torch.where(known, values - wanted, torch.zeros_like(values))[:, sp['burn_in']:]
        return (off ** 2).sum() / known[:, sp['burn_in']:].sum().clamp(min=1)

    def train_step(self) -> float:
        loss = self.loss(*self.sample())
        self.optimizer.zero_grad(set_to_none=True)
        loss.backward()
        self.optimizer.step()
        self.train_step_counter += 1
        if self.train_step_counter % int(self.spec['target_update_period']) == 0:
            self.target.load_state_dict(self.q_net.state_dict())
        return float(loss.detach())

    def train(self, num_iterations: int, initial_collect_steps: Optional[int] = None, collect_steps_per_iteration: int = 1,
              log_interval: int = 0) -> List[float]:
        """Collect, sample, train; ``initial_collect_steps`` defaults to one window."""
        self.collect(self.spec['window'] + 1 if initial_collect_steps is None else initial_collect_steps, epsilon=1.0)
        losses = []
        for it in range(num_iterations):
            self.collect(collect_steps_per_iteration)
            losses.append(self.train_step())
            if log_interval and (it + 1) % log_interval == 0:
                print('step = {0}: loss = {1}'.format(it + 1, losses[-1]))
        return losses

    @torch.no_grad()
    def evaluate(self, eval_env: PVDERVec) -> Dict[str, float]:
        """One greedy episode of every env of ``eval_env`` (auto_reset=False)."""
        assert not eval_env.auto_reset, "the evaluation env must not auto-reset"
        N, dev = eval_env.num_envs, eval_env.device
        c = eval_env._cfg()
        steps = -(-c.max_ksub // c.n_sub)
        if c.max_steps > 0:
            steps = min(steps, c.max_steps)
        state, ret = self.q_net.init_state(N), torch.zeros(N, dtype=torch.float64, device=dev)
        alive = torch.ones(N, dtype=torch.bool, device=dev)
        action, starts = torch.zeros(N, dtype=torch.uint8, device=dev), torch.ones(N, dtype=torch.bool, device=dev)
        eval_env.reset()
        out = eval_env.to_env_order(eval_env.out)
        for _ in range(steps):
            tokens = tokens_of(out[:N_OBS].t().contiguous(), action, out[11], starts)
            action.copy_(self._act(self.q_net.step(tokens, state, starts), 0.0))
            starts.fill_(False)
            eval_env.step(eval_env.to_lane_order(action) if eval_env.lane_io else action, return_tensors=False)
            out = eval_env.to_env_order(eval_env.out)
            ret += out[11].double() * alive
            alive &= out[12] == 0
        return {"average_return": float(ret.mean()), "min": float(ret.min()), "max": float(ret.max()), "steps": steps, "returns": ret}
