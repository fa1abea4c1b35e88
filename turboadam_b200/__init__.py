"""B200-native TurboAdam: packed-state optimizer step on hand-written sm_100a
kernels behind a C ABI (include/turboadam_b200.h), and the matrix operators
beside it (include/turboadam_b200_matrix.h)."""
from .matrix import linear_act, orthogonalize
from .muon import Muon
from .optimizer import TurboAdam, TurboAdamCommError

__version__ = "0.1.0"

__all__ = ["Muon", "TurboAdam", "TurboAdamCommError", "linear_act", "orthogonalize"]
