"""GGUF container: the reference's `Header` / `TensorInfo` / `Value` interface
(crates/ratchet-loader/src/gguf/gguf.rs) over the C ABI's rt_gguf_* entry points.

Parsing is host-only.  `Header.tensor(name, device)` uploads one tensor and brings it
into the library's layout (TensorInfo::read + ratchet_from_gguf, gguf.rs:63-84,118-142):
F32 / F16 as they are, Q8_0 through the device transcoder into Q8_0H (or Q8_0F), Q4_K as
raw super-blocks.
"""
from __future__ import annotations

import ctypes
import enum
from typing import Dict, List, Optional

import numpy as np

from . import _ffi
from .tensor import DType, Device, OperationError, Tensor, _stream_ptr, _torch, tensor_nbytes

DEFAULT_ALIGNMENT = 32  # gguf.rs:13


class GgmlDType(enum.IntEnum):
    """crates/ratchet-loader/src/lib.rs:35-101."""
    F32, F16, Q4_0, Q4_1, Q5_0, Q5_1, Q8_0, Q8_1 = 0, 1, 2, 3, 6, 7, 8, 9
    Q2K, Q3K, Q4K, Q5K, Q6K, Q8K = 10, 11, 12, 13, 14, 15

    def type_size(self) -> int:
        return int(_ffi.lib().rt_ggml_type_size(int(self)))

    def block_numel(self) -> int:
        return int(_ffi.lib().rt_ggml_block_numel(int(self)))

    def tensor_size(self, numel: int) -> int:
        return numel * self.type_size() // self.block_numel()


class ValueType(enum.IntEnum):
    """gguf.rs:183-214, ids :384-403."""
    U8, I8, U16, I16, U32, I32, F32, Bool, String, Array, U64, I64, F64 = range(13)


def _value(v: _ffi.GgufValue, fetch_elem=None):
    t = ValueType(v.type)
    if t in (ValueType.U8, ValueType.U16, ValueType.U32, ValueType.U64):
        return int(v.u64)
    if t in (ValueType.I8, ValueType.I16, ValueType.I32, ValueType.I64):
        return int(v.i64)
    if t in (ValueType.F32, ValueType.F64):
        return float(v.f64)
    if t == ValueType.Bool:
        return bool(v.u64)
    if t == ValueType.String:
        return ctypes.string_at(v.str, v.count).decode("utf-8", errors="replace")  # from_utf8_lossy, gguf.rs:180
    return [fetch_elem(i) for i in range(v.count)]


class TensorInfo:
    """gguf.rs:55-106."""

    def __init__(self, name: str, ggml_dtype: GgmlDType, shape, offset: int, size_in_bytes: int, index: int):
        self.name, self.ggml_dtype, self.shape = name, ggml_dtype, tuple(shape)
        self.offset, self._size, self.index = offset, size_in_bytes, index

    def size_in_bytes(self) -> int:
        return self._size

    def byte_range(self, tensor_data_offset: int) -> range:
        start = tensor_data_offset + self.offset
        return range(start, start + self._size)

    def __repr__(self):
        return f"TensorInfo({self.name!r}, {self.ggml_dtype.name}, {self.shape}, offset={self.offset})"


class Header:
    """gguf.rs:158-165: magic/version, metadata, tensor infos, tensor_data_offset."""

    def __init__(self, image: bytes):
        self._image = bytes(image)
        self._buf = ctypes.create_string_buffer(self._image, len(self._image))
        h = ctypes.c_void_p()
        st = _ffi.lib().rt_gguf_parse(self._buf, len(self._image), ctypes.byref(h))
        if st != _ffi.RT_OK:
            raise OperationError(st, "gguf: cannot parse the image")
        self._h = h
        L = _ffi.lib()
        self.version = int(L.rt_gguf_version(h))
        self.tensor_data_offset = int(L.rt_gguf_tensor_data_offset(h))
        self.metadata: Dict[str, object] = {}
        self.metadata_types: Dict[str, ValueType] = {}
        for i in range(L.rt_gguf_metadata_count(h)):
            key = ctypes.c_char_p()
            L.rt_gguf_metadata_key_at(h, i, ctypes.byref(key))
            v = _ffi.GgufValue()
            L.rt_gguf_metadata_get(h, key.value, ctypes.byref(v))
            name = key.value.decode("utf-8", errors="replace")
            self.metadata[name] = _value(v, lambda j, k=key.value: self._elem(k, j))
            self.metadata_types[name] = ValueType(v.type)
        self.tensor_infos: Dict[str, TensorInfo] = {}
        self.tensor_order: List[str] = []
        for i in range(L.rt_gguf_tensor_count(h)):
            ti = _ffi.GgufTensorInfo()
            L.rt_gguf_tensor_info_at(h, i, ctypes.byref(ti))
            name = ti.name.decode("utf-8", errors="replace")
            self.tensor_infos[name] = TensorInfo(name, GgmlDType(ti.ggml_dtype), [ti.shape[d] for d in range(ti.rank)],
                                                 int(ti.offset), int(ti.size_in_bytes), i)
            self.tensor_order.append(name)

    @staticmethod
    def read(image: bytes) -> "Header":
        """Header::read (gguf.rs:408-479)."""
        return Header(image)

    def _elem(self, key: bytes, i: int):
        v = _ffi.GgufValue()
        st = _ffi.lib().rt_gguf_metadata_array_get(self._h, key, i, ctypes.byref(v))
        if st != _ffi.RT_OK:
            raise OperationError(st, _ffi.lib().rt_gguf_error(self._h).decode())
        if ValueType(v.type) == ValueType.Array:
            raise OperationError(_ffi.RT_ERR_UNSUPPORTED, "nested arrays are not exposed element-wise")
        return _value(v)

    def get(self, key: str):
        """Metadata::get (gguf.rs:149-154)."""
        if key not in self.metadata:
            raise OperationError(_ffi.RT_ERR_INVALID_ARG, f"missing key {key}")
        return self.metadata[key]

    def tensor(self, name: str, device: Device, q8_dtype: DType = DType.Q8_0H, q4_0: bool = False) -> Tensor:
        """Header::tensor (gguf.rs:483-496).  The reference picks Q8_0H when the device has f16
        shaders (gguf.rs:130-136); every gfx950 does, so that is the default here.  Q4_0 tensors, on which the
        reference bails (gguf.rs:140), load with `q4_0` only."""
        if name not in self.tensor_infos:
            raise OperationError(_ffi.RT_ERR_INVALID_ARG, f"cannot find tensor info for {name}")
        if not device.is_gpu():
            raise OperationError(_ffi.RT_ERR_NO_DEVICE, "tensors are loaded to a GPU device")
        ti = self.tensor_infos[name]
        dst_dt = {GgmlDType.F32: DType.F32, GgmlDType.F16: DType.F16, GgmlDType.Q8_0: q8_dtype,
                  GgmlDType.Q4K: DType.Q4_K, GgmlDType.Q4_0: DType.Q4_0 if q4_0 else None}.get(ti.ggml_dtype)
        if dst_dt is None:
            raise OperationError(_ffi.RT_ERR_UNSUPPORTED, f"unsupported ggml dtype {ti.ggml_dtype.name}")
        numel = int(np.prod(ti.shape, dtype=np.int64)) if ti.shape else 1
        torch = _torch()
        dev = f"cuda:{device.ordinal}"
        dst = torch.empty(max(tensor_nbytes(dst_dt, numel), 16), dtype=torch.uint8, device=dev)
        staging = torch.empty(max(ti.size_in_bytes(), 16), dtype=torch.uint8, device=dev) \
            if ti.ggml_dtype in (GgmlDType.Q8_0, GgmlDType.Q4_0) else None
        st = _ffi.lib().rt_gguf_load_tensor(device.ctx, self._h, self._buf, len(self._image), ti.index, int(dst_dt),
                                            None if staging is None else ctypes.c_void_p(staging.data_ptr()),
                                            ctypes.c_void_p(dst.data_ptr()), _stream_ptr())
        if st != _ffi.RT_OK:
            raise OperationError(st, _ffi.lib().rt_last_error(device.ctx).decode())
        torch.cuda.current_stream().synchronize()  # the staging buffer and the image are released after this
        return Tensor(ti.shape, dst_dt, device, dst)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            _ffi.lib().rt_gguf_free(h)
            self._h = None
