"""KV cache held in 4 bits: quantised as it is written, read back, and attended to.

``Q4KVCache`` wraps the two device buffers of a cache (and its page table) as torch tensors and
runs the operators of ``libggmlc_b200.so`` on them (``gb_kv_q4_*``, include/ggmlc_b200.h, which
documents the format).  Every call runs on the current CUDA stream of the cache's device and
returns without waiting.  Calls may be captured by ``torch.cuda.graph``; a graph's scratch is its own,
so graphs may be replayed in any order and side by side.

    cache = Q4KVCache.empty(n_pages=64, n_kv_heads=8, page_len=256, head_dim=128,
                            pages=torch.tensor([[3, 7], [1, 5]], dtype=torch.int32, device="cuda"))
    cache.write(k, v, pos, slot)          # k, v [rows, 8, 128]; pos, slot int32 [rows] or ints
    o = cache.attend(q, pos, slot)        # q [rows, 32, 128]
    k, v = cache.read(pos, slot, torch.float16)

An int ``pos`` names consecutive positions pos, pos + 1, .. of one sequence (a prompt's chunk), an
int ``slot`` one sequence for all rows.
"""

from __future__ import annotations

import ctypes

import torch

from . import _runtime

try:
    from . import _kv_q4
except ImportError as e:
    raise ImportError("ggmlc_b200._kv_q4 is not built; build it with `python -m ggmlc_b200.build` "
                      "(g++ and torch's headers)") from e

_P, _I, _I64, _F, _SZ = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float,
                         ctypes.c_size_t)


class _Cache(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("n_pages", _I64), ("page_len", _I64), ("n_kv_heads", _I64),
                ("head_dim", _I64), ("pages", _P), ("n_slots", _I64), ("pages_per_slot", _I64)]


class _Rows(ctypes.Structure):
    _fields_ = [("n", _I64), ("pos", _P), ("pos0", _I64), ("slot", _P), ("slot0", _I64)]


_lib = _runtime.lib()
for _name, _args, _res in (
        ("gb_kv_q4_page_bytes", [_I64, _I64], _I64),
        ("gb_kv_q4_write", [_P, _P, _I, _P, _I64, _I64, _P, _I64, _I64, _P], _I),
        ("gb_kv_q4_read", [_P, _P, _I, _P, _P, _P], _I),
        ("gb_kv_q4_attend_workspace_bytes", [_P, _I64, _I64], _SZ),
        ("gb_kv_q4_attend", [_P, _P, _I, _P, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ, _P], _I),
        ("gb_kv_q4_attend_prefill", [_P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ,
                                     _P], _I),
        ("gb_kv_q4_error", [], _I),
        ("gb_kv_q4_clear_error", [], _I),
        ("gb_kv_q4_expire_waits", [_I], None)):
    getattr(_lib, _name).argtypes = _args
    getattr(_lib, _name).restype = _res


def page_bytes(page_len: int, head_dim: int) -> int:
    """Bytes of one head's page of page_len positions (a multiple of 16)."""
    n = int(_lib.gb_kv_q4_page_bytes(int(page_len), int(head_dim)))
    if n < 0:
        raise ValueError("page_len must be a positive multiple of 16 and head_dim of 32")
    return n


def error() -> int:
    """Non-zero once a bounded wait inside the attention of a chunk has run out on the current device
    (after about 2 s; that call's rows are NaN); waits for the device.  ``clear_error()`` resets it."""
    torch.cuda.synchronize()
    v = int(_lib.gb_kv_q4_error())
    if v < 0:
        raise RuntimeError(_lib.gb_last_error().decode())
    return v


def clear_error() -> None:
    torch.cuda.synchronize()
    if _lib.gb_kv_q4_clear_error() != 0:
        raise RuntimeError(_lib.gb_last_error().decode())


class Q4KVCache(_kv_q4.Cache):
    """K and V pools ``uint8 [n_pages, n_kv_heads, page_bytes]`` and, for a paged cache, the page
    table ``int32 [n_slots, pages_per_slot]``; without one, page ``slot`` is a sequence's window.

    ``write``, ``read`` and ``attend`` are the compiled binding's (bindings/kv_q4.cpp)."""

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_len: int, head_dim: int,
              pages: torch.Tensor | None = None, device: str | torch.device = "cuda"):
        """A cache of zeros."""
        shape = (n_pages, n_kv_heads, page_bytes(page_len, head_dim))
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, head_dim, pages)
