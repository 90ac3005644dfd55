from .lstm import FusedLSTM
from .gated import GatedCore
from .actor_critic import ActorNet, CriticNet, make_models

__all__ = ["FusedLSTM", "GatedCore", "ActorNet", "CriticNet", "make_models"]
