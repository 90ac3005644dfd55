from .lstm import FusedLSTM
from .gated import GatedCore
from .actor_critic import ActorNet, CriticNet, make_models, state_dtype

__all__ = ["FusedLSTM", "GatedCore", "ActorNet", "CriticNet", "make_models", "state_dtype"]
