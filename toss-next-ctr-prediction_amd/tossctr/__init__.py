"""tossctr -- MI355X-native DARE + QNN-alpha CTR training hot path (drop-in for the reference's
src/models/wrapper.py CTRModel and the src/train.py step), compute in libctrhip.so (gfx950 HIP)."""
from .arch import Arch
from .ops import (diff_attention, diff_attention_bwd, diff_attention_fwd, layer_norm, layer_norm_bwd, layer_norm_fwd,
                  newton_schulz)
from .optim import ArenaEMA, FusedAdamW, FusedMuon, build_ema
from .wrapper import CTRModel

__all__ = ["Arch", "CTRModel", "FusedAdamW", "FusedMuon", "ArenaEMA", "build_ema", "layer_norm", "layer_norm_fwd",
           "layer_norm_bwd", "diff_attention", "diff_attention_fwd", "diff_attention_bwd", "newton_schulz"]
