"""ctypes binding of ``libintent_amd.so`` (the C ABI in ``include/intent_amd.h``).

The reference binds natively compiled entries the same way: ``ctypes.CDLL``
plus one flat C symbol per entry with pointer / int64 extent slots
(python/intent/runtime/native_artifact.py:194-262, runtime/native.py:14-120).
There is no fallback: if the library is missing every call raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
import threading
from pathlib import Path

from .errors import INTENT_OK, NativeLibraryError, status_error

PACKAGE = Path(__file__).resolve().parent
# INTENT_AMD_LIBRARY names another build of the same library (the host-side
# AddressSanitizer build the sanitizer test loads); the in-tree build otherwise.
LIBRARY_PATH = Path(os.environ.get("INTENT_AMD_LIBRARY") or PACKAGE / "_lib" / "libintent_amd.so")
ABI_VERSION = 1

P = ctypes.c_void_p
I64 = ctypes.c_int64
INT = ctypes.c_int
SIZE = ctypes.c_size_t
F32 = ctypes.c_float

# Entry -> (argtypes, restype). Mirrors include/intent_amd.h.
SIGNATURES: dict[str, tuple[list, object]] = {
    "intent_amd_abi_version": ([], INT),
    "intent_amd_last_error": ([], ctypes.c_char_p),
    "intent_amd_last_kernel": ([], ctypes.c_char_p),
    "intent_amd_device_arch": ([INT, ctypes.c_char_p, I64], INT),
    "intent_w8a16_matmul": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P], INT),
    "intent_w4a16_matmul": ([P, I64, I64, I64, P, I64, I64, P, P, I64, I64, P, I64, P], INT),
    "intent_w4a16_gemv": ([P, I64, I64, I64, P, I64, I64, P, P, I64, I64, P, I64, P], INT),
    "intent_w4a16_gemm": ([P, I64, I64, I64, P, I64, I64, P, P, I64, I64, P, I64, P], INT),
    "intent_w8a16_matmul_workspace_size": ([I64, I64, I64], SIZE),
    "intent_w8a16_matmul_ws": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P, SIZE, P], INT),
    "intent_w4a16_gemm_workspace_size": ([I64, I64, I64, I64], SIZE),
    "intent_w4a16_gemm_ws": ([P, I64, I64, I64, P, I64, I64, P, P, I64, I64, P, I64, P, SIZE, P], INT),
    "intent_w4a16_matmul_workspace_size": ([I64, I64, I64, I64], SIZE),
    "intent_w4a16_matmul_ws": ([P, I64, I64, I64, P, I64, I64, P, P, I64, I64, P, I64, P, SIZE, P], INT),
    "intent_w8a8_gemm": ([P, I64, I64, I64, P, P, I64, I64, P, P, I64, P], INT),
    "intent_w8a8_gemm_workspace_size": ([I64, I64, I64], SIZE),
    "intent_w8a8_gemm_ws": ([P, I64, I64, I64, P, P, I64, I64, P, P, I64, P, SIZE, P], INT),
    "intent_i8_gemm_i32": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P], INT),
    "intent_i8_gemm_i32_kn": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P], INT),
    "intent_moe_route": ([P, I64, I64, I64, INT, P, P, P], INT),
    "intent_moe_align": ([P, I64, I64, I64, I64, P, I64, P, I64, P, P, P], INT),
    "intent_moe_gate_up_w4": ([P, I64, I64, I64, P, P, I64, I64, I64, P, P, P, I64, I64, I64, P, I64, P], INT),
    "intent_moe_down_w4": ([P, I64, P, P, I64, I64, I64, P, P, P, I64, I64, I64, I64, P, I64, P], INT),
    "intent_moe_combine": ([P, I64, P, I64, I64, P, I64, I64, P], INT),
    "intent_q8k_quantize": ([P, I64, I64, P, I64, P], INT),
    "intent_q4k_q8k_gemv": ([P, I64, I64, I64, P, P, P], INT),
    "intent_q4k_projection": ([P, I64, I64, I64, P, I64, P, P, P], INT),
    "intent_q4k_projection_noalloc": ([P, I64, I64, I64, P, I64, P, P], INT),
    "intent_fp8_groupwise_quantize": ([P, INT, I64, I64, I64, P, I64, P, I64, I64, P], INT),
    "intent_w4a8_gemm": ([P, I64, I64, I64, P, I64, I64, P, I64, P], INT),
    "intent_bitnet_int2_gemm": ([P, I64, I64, I64, P, I64, I64, P, I64, P], INT),
    "intent_mxfp8_gemm": ([P, I64, I64, I64, P, I64, P, I64, I64, P, I64, P, I64, P], INT),
    "intent_fp8_transpose": ([P, I64, I64, I64, P, I64, P], INT),
    "intent_scaled_fp8_gemm": ([P, I64, I64, I64, P, I64, I64, F32, F32, I64, INT, P, I64, P], INT),
    "intent_scaled_fp8_gemm_kn": ([P, I64, I64, I64, P, I64, I64, F32, F32, I64, INT, P, I64, P], INT),
    "intent_w4_sym_repack": ([P, I64, I64, I64, P, I64, I64, P, I64, P, P, I64, P], INT),
    "intent_w4a16_sym_gemv": ([P, I64, I64, I64, P, I64, I64, P, I64, P, I64, P], INT),
    "intent_w4a16_sym_gemm": ([P, I64, I64, I64, P, I64, I64, P, I64, P, I64, P], INT),
    "intent_f16_transpose": ([P, I64, I64, I64, P, I64, P], INT),
    "intent_quantized_gemm": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P, P, I64, P], INT),
    "intent_f16_transpose_batched": ([P, I64, I64, I64, I64, I64, P, I64, I64, P], INT),
    "intent_grouped_gemm": ([P, I64, I64, I64, P, I64, P, I64, P, I64, I64, I64, INT, P, I64, P], INT),
    "intent_grouped_gemm_kn": ([P, I64, I64, I64, P, I64, P, I64, I64, I64, INT, P, I64, P], INT),
    "intent_moe_expert_ffn_workspace_size": ([I64, I64, I64, I64], SIZE),
    "intent_moe_expert_ffn_workspace_size_for": ([I64, I64, I64, I64, I64], SIZE),
    "intent_moe_expert_ffn": ([P, I64, I64, I64, P, I64, P, I64, P, P, I64, P, P, I64, P, I64, P, SIZE, P], INT),
    "intent_f16_gemm": ([P, I64, I64, I64, P, I64, I64, INT, P, I64, P], INT),
    "intent_f16_gemm_kn": ([P, I64, I64, I64, P, I64, I64, INT, P, I64, P], INT),
    "intent_quantized_gemm_kn": ([P, I64, I64, I64, P, I64, I64, P, P, I64, P, P, I64, P], INT),
    "intent_nvfp4_quantize": ([P, I64, I64, I64, P, P, I64, P, P], INT),
    "intent_fp4_bf16_matmul": ([P, I64, I64, I64, P, I64, I64, P, I64, P], INT),
    "intent_fp8_gemm": ([P, I64, I64, I64, P, I64, I64, INT, P, I64, P], INT),
    "intent_deepgemm_fp8": ([P, I64, I64, I64, P, I64, P, I64, I64, P, I64, P, I64, P], INT),
    "intent_deepgemm_fp8_workspace_size": ([I64, I64, I64], SIZE),
    "intent_deepgemm_fp8_ws": ([P, I64, I64, I64, P, I64, P, I64, I64, P, I64, P, I64, P, SIZE, P], INT),
    "intent_moe_workspace_size": ([I64, I64, I64, I64, I64, I64], SIZE),
    "intent_moe_expert_ffn_w4": ([P, P, I64, I64, I64, I64, INT, P, P, P, P, P, P, I64, I64, P, P, SIZE, P, P, P],
                                 INT),
    "intent_i8_per_token_quantize": ([P, INT, I64, I64, I64, P, I64, P, P], INT),
    "intent_qk_norm_rope": ([P, I64, I64, I64, P, I64, I64, I64, P, P, F32, P, I64, I64, I64, INT, P, INT, P, I64, P,
                             I64, P], INT),
    "intent_paged_kv_append": ([P, I64, I64, I64, P, I64, I64, P, I64, I64, P, P, F32, P, I64, I64, I64, INT, P, P, INT,
                                INT, P, I64, P, I64, P, I64, P, I64, I64, I64, P, I64, P], INT),
    "intent_paged_attention": ([P, I64, I64, I64, INT, INT, P, I64, P, I64, P, I64, P, I64, I64, I64, I64, I64, P, I64,
                                I64, I64, P, P, F32, INT, I64, P, I64, P, SIZE, P], INT),
    "intent_paged_attention_workspace_size": ([I64, I64, I64, I64, I64, I64, I64], SIZE),
    "intent_paged_kv_append_int4": ([P, I64, I64, I64, P, I64, I64, P, I64, I64, P, P, F32, P, I64, I64, I64, INT, P, P,
                                     INT, P, I64, P, I64, P, I64, P, I64, I64, I64, P, I64, P], INT),
    "intent_paged_kv_read": ([INT, P, I64, P, I64, P, I64, P, I64, I64, I64, I64, I64, P, I64, INT, P, I64, P, I64, P], INT),
    "intent_biased_paged_attention": ([P, I64, I64, I64, INT, INT, P, I64, P, I64, P, I64, P, I64, I64, I64, I64, I64, P,
                                       I64, I64, I64, P, P, F32, INT, I64, F32, P, P, P, I64, P, SIZE, P], INT),
    "intent_biased_paged_attention_workspace_size": ([I64, I64, I64, I64, I64, I64, I64, INT], SIZE),
    "intent_amd_replay": ([INT, P, I64, P], INT),
    "intent_hbm_read_probe": ([P, I64, INT, INT, P, I64, P], INT),
    "intent_mfma_peak_probe": ([INT, I64, I64, P, P], INT),
}

_lock = threading.Lock()
_library: ctypes.CDLL | None = None


def library() -> ctypes.CDLL:
    """Load (once) and return the gfx950 library; raises if it is not built."""
    global _library
    if _library is not None:
        return _library
    with _lock:
        if _library is not None:
            return _library
        if not LIBRARY_PATH.exists():
            raise NativeLibraryError(
                f"{LIBRARY_PATH} is not built; run `python -m intent_amd.build` (hipcc, gfx950). "
                "There is no CPU fallback for the quantized-contraction kernels.")
        lib = ctypes.CDLL(str(LIBRARY_PATH))
        for name, (argtypes, restype) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError as error:
                raise NativeLibraryError(f"{LIBRARY_PATH} does not export {name}") from error
            fn.argtypes = argtypes
            fn.restype = restype
        version = lib.intent_amd_abi_version()
        if version != ABI_VERSION:
            raise NativeLibraryError(f"ABI version {version} != expected {ABI_VERSION}")
        _library = lib
        return lib


def last_error() -> str:
    raw = library().intent_amd_last_error()
    return raw.decode("utf-8", "replace") if raw else ""


def last_kernel() -> str:
    """The kernel variant the calling thread's latest launch dispatched to."""
    raw = library().intent_amd_last_kernel()
    return raw.decode("utf-8", "replace") if raw else ""


def call(entry: str, *arguments) -> None:
    """Invoke an int-status entry and raise the mapped exception on failure."""
    status = getattr(library(), entry)(*arguments)
    if status != INTENT_OK:
        raise status_error(status, entry, last_error())


class _Slots:
    """An entry that intent_amd_replay takes as slots: its number, and a packer of its arguments (ctypes
    converts some 30 of them one by one; packed they are one of four: a launch from Python 7.3 us, 8.4 before)."""

    def __init__(self, number: int, entry: str):
        types = SIGNATURES[entry][0][:-1]
        self.number = number
        self.count = len(types)
        self.entry = entry
        self._pack = struct.Struct("<" + "".join("f4x" if t is F32 else "q" for t in types)).pack

    def pack(self, arguments) -> bytes:
        try:
            return self._pack(*arguments)
        except OverflowError as error:  # no f32 holds the scalar
            raise ValueError(f"{self.entry}: {error}") from None


RECORDS = {entry: _Slots(number, entry)
           for number, entry in enumerate(("intent_qk_norm_rope", "intent_paged_kv_append", "intent_paged_attention",
                                           "intent_paged_kv_append_int4", "intent_paged_kv_read",
                                           "intent_biased_paged_attention"))}


def call_packed(entry: str, arguments: tuple, stream: int) -> None:
    """``call`` of one of the entries in RECORDS; null pointers are 0."""
    slots = RECORDS[entry]
    status = library().intent_amd_replay(slots.number, slots.pack(arguments), slots.count, stream)
    if status != INTENT_OK:
        raise status_error(status, entry, last_error())


class Record:
    """A call of an entry kept as slots: repeated for a stream without its arguments being converted again."""

    def __init__(self, entry: str, arguments: tuple):
        slots = RECORDS[entry]
        if len(arguments) != slots.count:
            raise TypeError(f"{entry} takes {slots.count} arguments before the stream, got {len(arguments)}")
        self.entry = entry
        self._number = slots.number
        self._count = slots.count
        self._slots = slots.pack(0 if a is None else a for a in arguments)
        self._replay = library().intent_amd_replay

    def __call__(self, stream: int) -> None:
        status = self._replay(self._number, self._slots, self._count, stream)
        if status != INTENT_OK:
            raise status_error(status, self.entry, last_error())


def device_arch(device: int) -> str:
    buf = ctypes.create_string_buffer(128)
    call("intent_amd_device_arch", device, buf, len(buf))
    return buf.value.decode()
