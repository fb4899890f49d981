from .qagent import BatchedQAgent  # noqa: F401
from .dqn import BatchedDQNAgent, QNetwork  # noqa: F401  (the TF-Agents DQN demo's loop, env and acting policy on the device)
from .sequence import BatchedSequenceDQNAgent, SequenceQNetwork  # noqa: F401  (DQN with a memory of the episode, on the operators of sequence_ops)
