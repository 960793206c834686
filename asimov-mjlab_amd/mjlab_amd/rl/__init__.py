from mjlab_amd.rl.memory import PolicyMemory
from mjlab_amd.rl.vecenv_wrapper import ObsDict, RslRlVecEnvWrapper

__all__ = ["ObsDict", "PolicyMemory", "RslRlVecEnvWrapper"]
