"""B200-native Cut Cross-Entropy: the ``cut_cross_entropy`` API over hand-written sm_100a CUDA."""

from .cce_utils import LinearCrossEntropyImpl
from .linear_cross_entropy import LinearCrossEntropy, linear_cross_entropy
from .linear_logits import linear_logits
from .sampling import linear_sample, sample_tokens
from .vocab_parallel import VocabParallelOptions

__all__ = [
    "LinearCrossEntropy",
    "LinearCrossEntropyImpl",
    "linear_cross_entropy",
    "linear_logits",
    "linear_sample",
    "sample_tokens",
    "VocabParallelOptions",
]

__version__ = "0.1.0"
