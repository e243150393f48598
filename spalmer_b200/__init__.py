"""B200-native routed micro-expert channel mixer for SPALMER.

Drop-in for ``spalmer.experts.MicroExpertChannelMixer`` (same constructor,
``forward`` contract and ``state_dict``), executed by hand-written sm_100a
kernels in ``libspx`` (``include/spx.h``).
"""

from spalmer_b200.config import MicroExpertsConfig
from spalmer_b200.experts import (
    B200ChannelBlock,
    B200MicroExpertChannelMixer,
    ChannelMixerOutput,
    ExpertPotentiationController,
    ExpertResidency,
    MicroExpertBank,
    MicroExpertChannelMixer,
    NativeExpertPrecisionError,
    RMSNorm,
    SurpriseRouter,
    SwiGLU,
    dispatch,
    rms_norm,
    route,
)
from spalmer_b200.token_mixer import B200DecoderLayer, LinearAttentionMixer
from spalmer_b200.token_ops import (
    add_rms_norm,
    add_rms_norm_mxfp8,
    linear_attention,
    linear_attention_status,
    linear_attention_step,
    rotary_embed,
    rotary_frequencies,
)

__all__ = [
    "B200ChannelBlock",
    "B200DecoderLayer",
    "B200MicroExpertChannelMixer",
    "ChannelMixerOutput",
    "ExpertPotentiationController",
    "ExpertResidency",
    "LinearAttentionMixer",
    "MicroExpertBank",
    "MicroExpertChannelMixer",
    "MicroExpertsConfig",
    "NativeExpertPrecisionError",
    "RMSNorm",
    "SurpriseRouter",
    "SwiGLU",
    "add_rms_norm",
    "add_rms_norm_mxfp8",
    "dispatch",
    "linear_attention",
    "linear_attention_status",
    "linear_attention_step",
    "rms_norm",
    "rotary_embed",
    "rotary_frequencies",
    "route",
]
