"""B200-native drop-in for the `ssd` package of Hprairie/Bi-Mamba2: the bidirectional SSD chunk scan operator
(`ssd.bi.ssd_combined.bimamba_chunk_scan_combined`) and the `ssd.modules.BiMamba2` layer built on it; and their causal
siblings for decoders (`ssd.uni.decay_attention`, `ssd.block_norm`, `ssd.modules.DecayDecoder`)."""
from ssd.modules import BiMamba2, Block, DecayAttention, DecayDecoder, Mamba2
from ssd.version import __version__

__all__ = ["BiMamba2", "Block", "DecayAttention", "DecayDecoder", "Mamba2", "__version__"]
