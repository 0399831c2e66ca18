"""B200-native (sm_100a) factored constant-Q transform.

Drop-in for the Flash-CQT API: ``OctCQT``, ``FusedOctCQT``, ``TrainableCQT``,
``SlicedCQT`` and ``Graphed``, all running on hand-written CUDA kernels behind
the C ABI of ``include/flash_cqt_b200.h``; plus ``HostPipeline`` for batches
that live in host memory (copies in both directions overlapped with the
transform), ``AdamW`` (the optimizer's step over many tensors, moments in 32 or
8 bits) and ``CoefCache`` (the newest slices of a set of streams in 8 bits).
"""
from .oct_cqt import OctCQT
from .sliced import SlicedCQT
from .graphed import Graphed
from .fused import FusedOctCQT
from .trainable import TrainableCQT
from .hostio import HostPipeline
from .optim import AdamW
from .coefcache import CoefCache

__all__ = ["OctCQT", "SlicedCQT", "Graphed", "FusedOctCQT", "TrainableCQT", "HostPipeline",
           "AdamW", "CoefCache"]
