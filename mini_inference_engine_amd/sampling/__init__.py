from .params import SamplingParams
from .rules import RuleInputs
from .sampler import Sampler
