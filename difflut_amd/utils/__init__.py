from .modules import (Dropout, GroupNorm, GroupSum, Linear, Linear8, RMSNorm, TokenEmbedding, beam_reorder, beam_step, cross_entropy,
                      sample)
from .optim import BankAdam
from .warnings import (ConfigurationWarning, CUDAWarning, DefaultValueWarning, DiffLUTWarning, PerformanceWarning,
                       configure_warnings, disable_all_warnings, disable_cuda_warnings, enable_all_warnings,
                       enable_strict_mode, suppress_warnings, warn_default_value)
