from .activations import ShiftedSoftplus
from .chain import (ChainAttention, ChainEmbedding, ChainEncoder, ChainEncoderLayer,
                    CounterDropout, GroupNormAct, chain_attention, dropout_add, group_norm_act)
from .cutoff import CosineCutoff, IdentityCutoff
from .delta import (ChainDelta, ChainDeltaEncoder, ChainDeltaLayer, RMSNormAdd, gated_delta,
                    rms_norm_add, scaled_embedding)
from .gradients import EnergyOut, GradientsOut, SumOut
from .losses import EnergyMSE, ForceMSE, ForceRMSE, Loss
from .mlp import MLP, init_xavier_uniform
from .prior import (Dihedral, FourierSeries, Harmonic, HarmonicAngles, HarmonicBonds,
                    Repulsion, StaticDihedral, StaticHarmonicAngles, StaticHarmonicBonds,
                    StaticRepulsion)
from .radial_basis import ExpNormalBasis, GaussianBasis
from .schnet import CFConv, InteractionBlock, SchNet, StandardSchNet

__all__ = ["ShiftedSoftplus", "CosineCutoff", "IdentityCutoff", "EnergyOut", "GradientsOut",
           "SumOut", "EnergyMSE", "ForceMSE", "ForceRMSE", "Loss", "MLP",
           "init_xavier_uniform", "GaussianBasis", "ExpNormalBasis", "CFConv",
           "InteractionBlock", "SchNet", "StandardSchNet", "Harmonic", "HarmonicBonds",
           "HarmonicAngles", "FourierSeries", "Dihedral", "Repulsion", "StaticHarmonicBonds",
           "StaticHarmonicAngles", "StaticDihedral", "StaticRepulsion",
           "ChainAttention", "ChainEmbedding", "ChainEncoder", "ChainEncoderLayer",
           "CounterDropout", "GroupNormAct", "chain_attention", "dropout_add",
           "group_norm_act", "ChainDelta", "ChainDeltaEncoder", "ChainDeltaLayer",
           "RMSNormAdd", "gated_delta", "rms_norm_add", "scaled_embedding"]
