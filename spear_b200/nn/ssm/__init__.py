from .layer import SelectiveSSM, SSMState

__all__ = ["SelectiveSSM", "SSMState"]
