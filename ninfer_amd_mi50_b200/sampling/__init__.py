from .params import SamplingParams
from .rules import TokenLogs, apply_rules
from .sampler import Sampler, check_params, sample_reference, uniform_draw

__all__ = ["SamplingParams", "Sampler", "TokenLogs", "apply_rules", "check_params", "sample_reference", "uniform_draw"]
