from .attention import TemporalDiffAttention, diff_attention  # noqa: F401
from .rotary import QKNormRotary, RotaryEncoder, qk_norm_rotary, rotary_encode, rotary_frequencies  # noqa: F401
from .time_encoder import TimeEncoder  # noqa: F401
