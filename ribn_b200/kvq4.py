"""The KV cache held in 4 bits: rows written into a paged arena, values read back, and attention over it.

A serving program keeps one arena per layer (:func:`empty_cache`, a torch uint8 tensor ``[pages][kv_heads][18 * head_dim]``,
16 tokens a page, 4.5 bits per value) beside its page tables.  Tensors lie on one CUDA device; every call is enqueued on that
device's current stream, allocates at most its result and its scratch through torch, and may be captured into a graph.  These
are the calls of ``include/ribn_b200.h`` (``ribn_b200_kvq4_*``), where the format and the rules are written down; there is no
CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import KVQ4_BF16, KVQ4_F16, KVQ4_F32, OK, KvQ4AttentionArgs, lib

PAGE_TOKENS = 16
_TYPES = {torch.float32: KVQ4_F32, torch.float16: KVQ4_F16, torch.bfloat16: KVQ4_BF16}


def empty_cache(pages: int, kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An arena of `pages` 16-token pages, all values zero."""
    if head_dim not in (64, 128, 256) or pages <= 0 or kv_heads <= 0:
        raise ValueError("an arena has pages, kv heads and a head_dim of 64, 128 or 256")
    return torch.zeros((pages, kv_heads, 18 * head_dim), dtype=torch.uint8, device=device)


def _refuse(what: str):
    buf = C.create_string_buffer(1024)
    lib().ribn_b200_op_last_error(buf, len(buf))
    raise RuntimeError(f"ribn_b200 {what} failed: {buf.value.decode(errors='replace')}")


def _arena(cache: torch.Tensor):
    shape = cache.shape
    if cache.dtype is not torch.uint8 or len(shape) != 3 or not cache.is_cuda or not cache.is_contiguous() or shape[2] % 18:
        raise ValueError("cache must be a contiguous uint8 CUDA tensor [pages][kv_heads][18 * head_dim]")
    return shape[0], shape[1], shape[2] // 18, cache.get_device()


def _rows(name: str, x: torch.Tensor, heads: int, head_dim: int, device: int, rows: int | None = None, dtype=None):
    """A [rows][heads][head_dim] tensor whose rows are whole; the values from one row to the next."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim or (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}][{heads}][{head_dim}]: got {list(shape)}")
    if x.get_device() != device or x.dtype not in _TYPES or (dtype is not None and x.dtype is not dtype):
        raise ValueError(f"{name} must be float32, float16 or bfloat16, as its fellows are, on CUDA device {device}: got {x.dtype} on {x.device}")
    if shape[0] and (stride[2] != 1 or (heads > 1 and stride[1] != head_dim)):
        raise ValueError(f"{name}: the heads of a row must lie side by side")
    if shape[0] > 1 and stride[0] < heads * head_dim:
        raise ValueError(f"{name}: rows overlap")
    return stride[0]


def _ints(name: str, x: torch.Tensor, shape: tuple, device: int):
    """An int32 tensor of this shape whose last dimension is contiguous; its address."""
    if x.dtype is not torch.int32 or x.shape != shape or x.get_device() != device or (x.stride()[-1] != 1 and x.numel()):
        raise ValueError(f"{name} must be an int32 tensor of shape {list(shape)} on CUDA device {device}, its last dimension contiguous: "
                         f"got {x.dtype} {list(x.shape)} on {x.device}")
    return x.data_ptr()


_MOST, _MOST_KEYS = 2 ** 31 - 1, 2 ** 31 - 1 - PAGE_TOKENS


def _size(x: int, most: int) -> int:
    """A size for the C call, whose fields have 32 bits: one over `most` says what `most` says; a negative one is refused there."""
    return -1 if x < 0 else min(x, most)


# the stream as a number, without a Stream object around it, which takes longer to make than a small call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises rows k, v [rows][kv_heads][head_dim] into the arena at slots[row] = page * 16 + token.  A row with a slot outside
    of the arena (-1: padding) is not written.  The slots of one call are distinct.  NaN counts as zero, magnitudes over 7,168
    saturate.  A cache holds bytes: no gradient passes through it."""
    pages, kv_heads, head_dim, device = _arena(cache)
    k_stride = _rows("k", k, kv_heads, head_dim, device)
    rows = k.shape[0]
    v_stride = _rows("v", v, kv_heads, head_dim, device, rows, k.dtype)
    at = _ints("slots", slots, (rows,), device)
    if lib().ribn_b200_kvq4_append(device, _raw_stream(device), cache.data_ptr(), pages, kv_heads, head_dim, _TYPES[k.dtype], k.data_ptr(),
                                   k_stride, v.data_ptr(), v_stride, at, rows) != OK:
        _refuse("kvq4_append")


def read(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """(k, v) [rows][kv_heads][head_dim]: the cached values at slots[row], which float16 and float32 hold exactly; zeros where a slot
    lies outside of the arena."""
    pages, kv_heads, head_dim, device = _arena(cache)
    rows = slots.shape[0] if slots.dim() == 1 else -1
    at = _ints("slots", slots, (rows,), device)
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    # (with strides given it is made in two thirds of the time)
    shape, strides, where = (rows, kv_heads, head_dim), (kv_heads * head_dim, head_dim, 1), cache.device
    k, v = torch.empty_strided(shape, strides, dtype=dtype, device=where), torch.empty_strided(shape, strides, dtype=dtype, device=where)
    if lib().ribn_b200_kvq4_read(device, _raw_stream(device), cache.data_ptr(), pages, kv_heads, head_dim, _TYPES[dtype], at, rows,
                                 k.data_ptr(), v.data_ptr()) != OK:
        _refuse("kvq4_read")
    return k, v


def attention(cache: torch.Tensor, q: torch.Tensor, page_tables: torch.Tensor, lengths: torch.Tensor, cu_rows: torch.Tensor, *,
              max_rows: int, max_keys: int, window: int = 0, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal grouped-query attention over the arena: rows [cu_rows[s], cu_rows[s + 1]) of q [rows][q_heads][head_dim] are the last
    rows of sequence s, which has lengths[s] keys (these rows' own, already appended, among them) in the pages page_tables[s].
    Row i of n sits at position lengths[s] - n + i and sees the keys up to its own, with window > 0 the last `window` of those.

    Probabilities of float32 rows are held as pairs of binary16, of float16 and bfloat16 ones as one: float16 results are up to 1.3 times as far
    from exact ones as their own rounding.  A query that is not finite makes its row NaN where it sees a key.

    Rows that see no key get zeros, rows behind the last sequence stay as they are in `out` (zeros in a new one).  `max_rows` is
    the most rows of a sequence; `max_keys`, about the longest length, decides how the work is split and no result but for its last bits (below
    a true length of more than 32,768, sums of float16 rows lose up to 2^-24 for every 16 keys).  `out` does not overlap `q`.
    `scale` defaults to head_dim ** -0.5.  There is no backward pass: a `q` or `out` that requires a gradient is refused while gradients
    are recorded.  Returns `out`, of q's type."""
    pages, kv_heads, head_dim, device = _arena(cache)
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % kv_heads:
        raise ValueError(f"q must be [rows][q_heads][{head_dim}], q_heads a multiple of the cache's {kv_heads}")
    rows, q_heads, _ = q.shape
    q_stride = _rows("q", q, q_heads, head_dim, device)
    if page_tables.dim() != 2:
        raise ValueError("page_tables must be [sequences][pages of the longest]")
    sequences, width = page_tables.shape
    tables, at_lengths = _ints("page_tables", page_tables, (sequences, width), device), _ints("lengths", lengths, (sequences,), device)
    at_rows = _ints("cu_rows", cu_rows, (sequences + 1,), device)
    if scale is not None and not 1.2e-38 <= abs(scale) <= 3.4e38:   # zero would stand for the default
        raise ValueError("scale must be a float32 number other than zero")
    if (q.requires_grad or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("attention over a 4-bit cache has no backward pass: call it under torch.no_grad() or with detached tensors")
    if out is None:
        out = torch.zeros((rows, q_heads, head_dim), dtype=q.dtype, device=q.device)
    out_stride = _rows("out", out, q_heads, head_dim, device, rows, q.dtype)
    if not (0 <= max_rows <= rows and 0 <= max_keys <= _MOST_KEYS and 0 <= window <= _MOST):   # (one test in the common case, 1 us less)
        max_rows, max_keys, window = _size(max_rows, rows), _size(max_keys, _MOST_KEYS), _size(window, _MOST)
    args = KvQ4AttentionArgs(cache.data_ptr(), pages, q.data_ptr(), out.data_ptr(), tables, at_lengths, at_rows, None, 0, q_stride, out_stride,
                             page_tables.stride(0), _TYPES[q.dtype], q_heads, kv_heads, head_dim, width, sequences, rows,
                             max_rows, max_keys, window, scale or 0.0, 0)
    library = lib()
    need = library.ribn_b200_kvq4_workspace(args)
    if need:
        scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = scratch.data_ptr(), need
    if library.ribn_b200_kvq4_attention(device, _raw_stream(device), args) != OK:
        _refuse("kvq4_attention")
    return out
