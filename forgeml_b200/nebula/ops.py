"""Thin launch wrappers for the Nebula decode-step kernels (C ABI neb_*).

All take device tensors, launch on the current stream of their device and
raise on a nonzero status; none allocates except where an output is created.
The kv4_* wrappers (cache in 4 bits, ``cache.KV4Pool``) also check their
arguments (ValueError) and select the pool's device.
"""

from __future__ import annotations

import functools
import math

import torch

from forgeml_b200 import _native


def _stream(t: torch.Tensor) -> int:
    return _native.stream_ptr(t.device)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
              slot_of: torch.Tensor, start_pos: torch.Tensor) -> None:
    """pool[slot_of[b], h, start_pos[b]+t, :] = kv[b, t, h, :] (k, v: [B,T,H,D] views)."""
    b, t, h, d = k.shape
    max_seq = k_pool.shape[2]
    _native.call(
        "neb_kv_append", k.data_ptr(), _native.strides4(k), v.data_ptr(), _native.strides4(v),
        k_pool.data_ptr(), v_pool.data_ptr(), slot_of.data_ptr(), start_pos.data_ptr(),
        b, t, h, d, max_seq, _native.dtype_code(k.dtype), _stream(k),
    )


def attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, slot_of: torch.Tensor,
              start_pos: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Masked attention of q [B,T,H,D] over the cached prefix; returns [B,T,H*D]."""
    b, t, h, d = q.shape
    if out is None:
        out = torch.empty((b, t, h * d), dtype=q.dtype, device=q.device)
    _native.call(
        "neb_attention", q.data_ptr(), _native.strides4(q), k_pool.data_ptr(), v_pool.data_ptr(),
        slot_of.data_ptr(), start_pos.data_ptr(), out.data_ptr(), b, t, h, d, k_pool.shape[2], k_pool.shape[0],
        1.0 / math.sqrt(d), _native.dtype_code(q.dtype), _stream(q),
    )
    return out


# The kv4_* wrappers run once per layer and step, outside captured graphs too, so
# their checks are plain attribute comparisons and their strides' arrays are kept
# by value.
_I32 = torch.int32
_get_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _raw_stream(index: int) -> int:
    return _get_stream(index) if _get_stream is not None else torch.cuda.current_stream(index).cuda_stream


@functools.lru_cache(maxsize=1024)
def _kv4_strides(s0: int, s1: int, s2: int):
    return _native.strides4((s0, s1, s2, 1))


def _kv4_call(pool, name: str, *args) -> None:
    """One C call on the pool's device and its current stream."""
    index = pool.device.index
    if torch.cuda.current_device() == index:
        _native.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _native.call(name, *args, _raw_stream(index))


def _kv4_table(pool, name: str, t: torch.Tensor) -> int:
    """Check a batch's slot or position table; returns its length."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor")
    if t.device != pool.device:
        raise ValueError(f"{name} must be on the pool's device")
    return t.shape[0]


def _kv4_tables(pool, slot_of: torch.Tensor, start_pos: torch.Tensor | None) -> int:
    """Check a batch's tables; returns the batch size."""
    batch = _kv4_table(pool, "slot_of", slot_of)
    if start_pos is not None and _kv4_table(pool, "start_pos", start_pos) != batch:
        raise ValueError("start_pos must hold one entry per request")
    if batch == 0:
        raise ValueError("the batch must not be empty")
    return batch


def _kv4_rows(pool, name: str, x: torch.Tensor, batch: int):
    """Check rows [B, T, heads, head_dim]; returns T, heads and the strides' array."""
    if not isinstance(x, torch.Tensor) or x.dim() != 4:
        raise ValueError(f"{name} must be a tensor [B, T, heads, head_dim]")
    if x.dtype is not pool.dtype or x.device != pool.device:
        raise ValueError(f"{name} must match the pool's device and dtype")
    b, t, heads, d = x.shape
    if b != batch or t == 0 or d != pool.head_dim:
        raise ValueError(f"bad {name} shape {tuple(x.shape)}")
    s0, s1, s2, s3 = x.stride()
    if s3 != 1 and d > 1:
        raise ValueError(f"{name} needs unit stride in the head dimension")
    if t > pool.max_seq_len:
        raise ValueError("more rows than the pool's max_seq_len")
    return t, heads, _kv4_strides(s0, s1, s2)


def kv4_append(k: torch.Tensor, v: torch.Tensor, pool, slot_of: torch.Tensor, start_pos: torch.Tensor) -> None:
    """Quantise k and v [B,T,H,D] (views with unit innermost stride) into rows
    start_pos[b] .. start_pos[b]+T-1 of slot slot_of[b] of a ``KV4Pool``.

    The requests of a batch hold distinct slots: where a later request's rows
    overlap an earlier one's in the same slot, the earlier one's are kept and
    the device error word's bit 4 is raised, as for a slot or position outside
    the pool, whose rows are not written."""
    b = _kv4_tables(pool, slot_of, start_pos)
    t, heads, ks = _kv4_rows(pool, "k", k, b)
    vt, v_heads, vs = _kv4_rows(pool, "v", v, b)
    if heads != pool.heads:
        raise ValueError(f"bad k shape {tuple(k.shape)}")
    if v_heads != heads or vt != t:
        raise ValueError(f"bad v shape {tuple(v.shape)}")
    _kv4_call(pool, "neb_kv4_append", k.data_ptr(), ks, v.data_ptr(), vs, pool.handle, slot_of.data_ptr(),
              start_pos.data_ptr(), b, t)


def kv4_read(pool, slot_of: torch.Tensor, count: int, *, start_pos: torch.Tensor | None = None,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The numbers that rows start_pos[b] .. start_pos[b]+count-1 (from row 0
    without ``start_pos``) of slot slot_of[b] stand for, rounded to the pool's
    dtype: keys and values [B,H,count,D].  Rows of a slot or position outside
    the pool come back as zeros and raise the device error word's bit 4."""
    b = _kv4_tables(pool, slot_of, start_pos)
    if not isinstance(count, int) or isinstance(count, bool) or not 0 < count <= pool.max_seq_len:
        raise ValueError("count must be an integer in 1..max_seq_len")
    shape = (b, pool.heads, count, pool.head_dim)
    if out is None:
        ko = torch.empty(shape, dtype=pool.dtype, device=pool.device)
        vo = torch.empty_like(ko)
    else:
        ko, vo = out
        for x in (ko, vo):
            if not isinstance(x, torch.Tensor) or tuple(x.shape) != shape or x.dtype is not pool.dtype \
                    or x.device != pool.device or not x.is_contiguous():
                raise ValueError(f"out must be two contiguous {shape} tensors of the pool's dtype and device")
    _kv4_call(pool, "neb_kv4_read", pool.handle, slot_of.data_ptr(),
              start_pos.data_ptr() if start_pos is not None else None, count, ko.data_ptr(), vo.data_ptr(), b)
    return ko, vo


def kv4_attention(q: torch.Tensor, pool, slot_of: torch.Tensor, start_pos: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Masked attention of q [B,T,QH,D] over the quantised prefix: query t of
    request b sits at position start_pos[b]+t and attends rows 0 up to its own.
    QH is a multiple of the pool's heads; query head h reads head
    h // (QH // heads).  Returns [B,T,QH*D].  Scores, their maximum and the sums
    are held in fp32; weights go as 16-bit (bf16) or 23-bit integers, for more
    than 8 query rows of a head in 16-bit types as fp16 (include/forgeml_b200.h).
    A slot or position outside the pool gives zeros and raises the device
    error word's bit 4."""
    b = _kv4_tables(pool, slot_of, start_pos)
    t, qh, qs = _kv4_rows(pool, "q", q, b)
    if qh == 0 or qh % pool.heads:
        raise ValueError(f"bad q shape {tuple(q.shape)}")
    shape = (b, t, qh * pool.head_dim)
    if out is None:
        out = torch.empty(shape, dtype=pool.dtype, device=pool.device)
    elif tuple(out.shape) != shape or out.dtype is not q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {shape} tensor of q's dtype and device")
    need = pool.workspace_bytes(b, t, qh)
    ws = torch.empty(need, dtype=torch.uint8, device=pool.device) if need else None
    _kv4_call(pool, "neb_kv4_attention", q.data_ptr(), qs, pool.handle, slot_of.data_ptr(), start_pos.data_ptr(),
              out.data_ptr(), b, t, qh, pool.scale, ws.data_ptr() if need else None, need)
    return out


def embed(tokens: torch.Tensor, start_pos: torch.Tensor, tok_emb: torch.Tensor, pos_emb: torch.Tensor,
          out: torch.Tensor | None = None) -> torch.Tensor:
    b, t = tokens.shape
    hidden = tok_emb.shape[1]
    if out is None:
        out = torch.empty((b, t, hidden), dtype=tok_emb.dtype, device=tok_emb.device)
    _native.call(
        "neb_embed", tokens.data_ptr(), start_pos.data_ptr(), tok_emb.data_ptr(), pos_emb.data_ptr(),
        out.data_ptr(), b, t, hidden, tok_emb.shape[0], pos_emb.shape[0],
        _native.dtype_code(tok_emb.dtype), _stream(tok_emb),
    )
    return out


def argmax(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Row-wise argmax of a [rows, cols] view (unit column stride)."""
    rows, cols = logits.shape
    if logits.stride(1) != 1:
        raise ValueError("argmax needs unit column stride")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    _native.call(
        "neb_argmax", logits.data_ptr(), logits.stride(0), rows, cols, out.data_ptr(),
        _native.dtype_code(logits.dtype), _stream(logits),
    )
    return out


def add(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(a)
    _native.call("neb_add", a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(),
                 _native.dtype_code(a.dtype), _stream(a))
    return out
