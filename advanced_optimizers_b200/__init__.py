"""B200-native (sm_100a) optimizer step for the adv_optm optimizers.

Drop-in classes with the constructor arguments, param-group keys and state
layout of adv_optm 2.5.4; the step runs in hand-written CUDA kernels through
the C ABI in include/advopt.h (libadvopt.so, built in-tree).
"""
from .optim import *  # noqa: F401,F403
from .optim import __all__ as _optim_all
from .distributed import ShardedOptimizer
from .dropout import philox_dropout
from .fp8 import Fp8Blocks, check_fp8_errors, fp8_linear, fp8_matmul, quantize_fp8

__version__ = "0.1.0"
reference_version = "2.5.4"
__all__ = list(_optim_all) + ["ShardedOptimizer", "philox_dropout", "Fp8Blocks", "quantize_fp8", "fp8_matmul",
                               "fp8_linear", "check_fp8_errors"]
