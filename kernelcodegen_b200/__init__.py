"""B200 (sm_100a) kernels for the operators KernelCodeGen generates (fused matmul+ReLU and FMHA), the standalone
softmax, transpose and batched product, and attention for training with the norm and rotation of its queries and
keys, behind a C-ABI (`include/kcg_capi.h`)."""
from . import capi  # noqa: F401

__all__ = ["capi", "ops"]


def __getattr__(name):
    if name == "ops":
        import importlib

        return importlib.import_module(".ops", __name__)
    raise AttributeError(name)
