"""ratchet_amd: MI355X (gfx950) backend for ratchet-core's Matmul operator.

The product is libratchet_hip.so (C ABI in include/ratchet_hip.h, sources in
ratchet_amd/csrc).  This package is the thin host-side mirror of the
reference's operator interface used to drive it from Python.
"""
from ._ffi import LIB_PATH, lib  # noqa: F401
from .tensor import (DType, Device, DeviceRequest, InvariantError, Matmul, OperationError, Quantization,  # noqa: F401
                     Quantizer, Sequences, Tensor, dequantize, tensor_nbytes, transcode_gguf_q4_0, transcode_gguf_q8_0)
from . import gguf  # noqa: F401,E402  (Header / TensorInfo / GgmlDType: the GGUF container)
from . import nn  # noqa: F401,E402  (Linear, MLP, KVCache, SelfAttention: the module harness)
