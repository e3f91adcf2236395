"""Operator entry points on torch CUDA tensors (one per reference Metal
pipeline; MetalManager.swift:43-49).  Tensors carry device memory only: each
function passes raw pointers to libqwen_b200.so and enqueues on the current
torch stream.
"""
from __future__ import annotations

import struct
from ctypes import byref

import torch

from ._lib import QWEN_DTYPE_BF16, QWEN_DTYPE_F16, PagedKVStruct, check, lib

HIDDEN, INTER, HEADS, KV_DIM, HEAD_DIM = 1536, 8960, 12, 256, 128
VOCAB, ACTUAL_VOCAB = 151936, 151666


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def gemv_q4_0(packed: torch.Tensor, scales: torch.Tensor, x: torch.Tensor,
              bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """gemv_q4_0 (matmul.metal:9-73): y = half((W_deq x) + bias)."""
    k = x.numel()
    n = scales.numel() * 32 // k
    y = out if out is not None else torch.empty(n, dtype=torch.float16, device=x.device)
    check(lib().qwen_gemv_q4_0(_ptr(packed), _ptr(scales), _ptr(x), _ptr(y), k, _ptr(bias), n,
                               _stream()))
    return y


def gemv_fp16(w: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """gemv_fp16 (matmul.metal:75-113)."""
    n, k = w.shape
    y = out if out is not None else torch.empty(n, dtype=torch.float16, device=x.device)
    check(lib().qwen_gemv_fp16(_ptr(w), _ptr(x), _ptr(y), k, n, _stream()))
    return y


def gemm_q4_0_batched(packed: torch.Tensor, scales: torch.Tensor, x: torch.Tensor,
                      bias: torch.Tensor | None = None) -> torch.Tensor:
    """gemv_q4_0 (matmul.metal:9-73) for every row of x [n_batch][k] at once on
    the tcgen05 tensor cores: y [n_batch][n_rows]."""
    nb, k = x.shape
    n = scales.numel() * 32 // k
    y = torch.empty((nb, n), dtype=torch.float16, device=x.device)
    check(lib().qwen_gemm_q4_0_batched(_ptr(packed), _ptr(scales), _ptr(x), _ptr(y), k, _ptr(bias),
                                       n, nb, _stream()))
    return y


def gemm_fp16_batched(w: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """gemv_fp16 (matmul.metal:75-113) for every row of x [n_batch][k] at once."""
    n, k = w.shape
    nb = x.shape[0]
    y = torch.empty((nb, n), dtype=torch.float16, device=x.device)
    check(lib().qwen_gemm_fp16_batched(_ptr(w), _ptr(x), _ptr(y), k, n, nb, _stream()))
    return y


def rms_norm_q4(x: torch.Tensor, gamma: torch.Tensor) -> torch.Tensor:
    """rms_norm_q4 (rmsnorm.metal:9-46)."""
    out = torch.empty_like(x)
    check(lib().qwen_rms_norm_q4(_ptr(x), _ptr(gamma), _ptr(out), _stream()))
    return out


def apply_rope_q4(vec: torch.Tensor, n_heads: int, seq_len: torch.Tensor) -> torch.Tensor:
    """apply_rope_q4 (rope.metal:12-39), in place; seq_len is a 1-element uint32/int32 tensor."""
    check(lib().qwen_apply_rope_q4(_ptr(vec), n_heads, _ptr(seq_len), _stream()))
    return vec


def write_kv_cache(k, v, k_cache, v_cache, seq_len, max_ctx: int) -> None:
    """write_kv_cache (attention.metal:67-84)."""
    check(lib().qwen_write_kv_cache(_ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ptr(seq_len),
                                    max_ctx, _stream()))


def attention_scores(q, k_cache, scores, seq_len, max_ctx: int) -> None:
    check(lib().qwen_attention_scores(_ptr(q), _ptr(k_cache), _ptr(scores), _ptr(seq_len), max_ctx,
                                      _stream()))


def softmax(scores, seq_len) -> None:
    check(lib().qwen_softmax(_ptr(scores), _ptr(seq_len), _stream()))


def attn_weighted_sum(scores, v_cache, out, seq_len) -> None:
    check(lib().qwen_attn_weighted_sum(_ptr(scores), _ptr(v_cache), _ptr(out), _ptr(seq_len),
                                       _stream()))


def residual_add(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    out = out if out is not None else torch.empty_like(a)
    check(lib().qwen_residual_add(_ptr(a), _ptr(b), _ptr(out), a.numel(), _stream()))
    return out


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """swiglu (activations.metal:9-27), in place on gate."""
    check(lib().qwen_swiglu(_ptr(gate), _ptr(up), gate.numel(), _stream()))
    return gate


def attention_decode(q, k_cache, v_cache, seq_len, max_ctx: int) -> torch.Tensor:
    """Fused split-K GQA decode attention over a reference-layout cache."""
    out = torch.empty(HIDDEN, dtype=torch.float16, device=q.device)
    check(lib().qwen_attention_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                      _ptr(seq_len), max_ctx, _stream()))
    return out


def attention_decode_batched(q, k_cache, v_cache, seq_len, max_ctx: int) -> torch.Tensor:
    """attention_decode for every sequence: q [n][1536], caches [n][max_ctx][256],
    seq_len [n] (device uint32/int32)."""
    n = q.shape[0]
    out = torch.empty((n, HIDDEN), dtype=torch.float16, device=q.device)
    check(lib().qwen_attention_decode_batched(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                              _ptr(seq_len), n, max_ctx, _stream()))
    return out


def dequant_q4(packed: torch.Tensor, scales: torch.Tensor, n_weights: int) -> torch.Tensor:
    out = torch.empty(n_weights, dtype=torch.float32, device=packed.device)
    check(lib().qwen_dequant_q4(_ptr(packed), _ptr(scales), n_weights, _ptr(out), _stream()))
    return out


def quantize_q4(w: torch.Tensor):
    """packAndSave4Bit (QwenPipelines.swift:97-145) on the device."""
    w = w.contiguous().float().view(-1)
    nb = (w.numel() + 31) // 32
    packed = torch.empty(nb * 16, dtype=torch.uint8, device=w.device)
    scales = torch.empty(nb, dtype=torch.float16, device=w.device)
    check(lib().qwen_quantize_q4(_ptr(w), w.numel(), _ptr(packed), _ptr(scales), _stream()))
    return packed, scales


def sample(logits: torch.Tensor, temperature: float, top_p: float,
           u24: torch.Tensor | None = None, vocab: int = ACTUAL_VOCAB,
           scratch: torch.Tensor | None = None) -> torch.Tensor:
    """extractNextTokenID (InferenceEngine.swift:273-368) on the device.

    logits: [n_seq, row_stride] fp16; u24: [n_seq] 24-bit uniforms (int32).
    scratch: device bytes from sample_scratch(n_seq) (qwen_sample_scratch: one
    sequence over every SM); None runs qwen_sample (one cluster per sequence)."""
    if logits.dim() == 1:
        logits = logits.view(1, -1)
    n_seq, stride = logits.shape
    out = torch.empty(n_seq, dtype=torch.int32, device=logits.device)
    if scratch is None:
        check(lib().qwen_sample(_ptr(logits), n_seq, stride, vocab, temperature, top_p, _ptr(u24),
                                _ptr(out), _stream()))
    else:
        check(lib().qwen_sample_scratch(_ptr(logits), n_seq, stride, vocab, temperature, top_p,
                                        _ptr(u24), _ptr(out), _ptr(scratch), _stream()))
    return out


def sample_scratch(n_seq: int, device) -> torch.Tensor | None:
    """Zeroed scratch for sample(..., scratch=...) (None when n_seq needs none)."""
    n = lib().qwen_sample_scratch_bytes(n_seq)
    return torch.zeros(n, dtype=torch.uint8, device=device) if n else None


def uniform24(seed: int, sequence: int, step: int) -> int:
    return lib().qwen_uniform24(seed, sequence, step)


# ---------------------------------------------------------- paged cache -----
# A decode step's kernels take 2 to 25 us, and torch's and ctypes' share of a call as
# much: these wrappers read each property of a tensor once, pass plain numbers on and
# take memory with new_empty(sizes) (1.3 us; torch.empty(size, dtype=, device=) 1.6 to 2.4).
_PAGED_KV = struct.Struct("=4Q3q7Ii")   # qwen_paged_kv, half a microsecond faster than field by field
_DTYPES = {torch.float16: QWEN_DTYPE_F16, torch.bfloat16: QWEN_DTYPE_BF16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") \
    else lambda index: torch.cuda.current_stream(index).cuda_stream
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") \
    else torch.cuda.current_device
_UINT32 = 0xFFFFFFFF   # ctypes would cut a larger number to its low 32 bits
_workspace_bytes: dict = {}   # by sizes: the library's answers are functions of nothing else


class PagedKV:
    """One layer's paged key/value cache (qwen_paged_kv) over the caller's tensors.

    k_pages, v_pages: [n_pages, page_size, n_kv_heads, head_dim], fp16 or bf16, any
    (equal) strides with the head's elements adjacent: head-major pages are
    `pool.transpose(1, 2)`.  page_table: int32 [n_seq, max_pages], the pool page of
    each sequence's page.  bounds: [n_pages, 2, n_kv_heads, head_dim], the least and
    largest stored key of each page (kept by rope_append_paged, read by
    select_pages); None keeps none.  The object holds references to the tensors and
    reads nothing of their contents; their shapes and addresses must not change."""

    __slots__ = ("k_pages", "v_pages", "page_table", "bounds", "dtype", "device", "index", "n_seq",
                 "n_kv_heads", "head_dim", "page_size", "sizes", "ref", "_struct")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 bounds: torch.Tensor | None = None):
        dtype, index = k_pages.dtype, k_pages.get_device()
        if dtype not in _DTYPES:
            raise ValueError(f"k_pages must be float16 or bfloat16, not {dtype}")
        if index < 0:
            raise ValueError("expected a CUDA tensor")
        shape, st = k_pages.shape, k_pages.stride()
        if len(shape) != 4:
            raise ValueError("k_pages must be [n_pages, page_size, n_kv_heads, head_dim]")
        if v_pages.shape != shape or v_pages.stride() != st or v_pages.dtype is not dtype:
            raise ValueError("k_pages and v_pages must have the same shape, strides and dtype")
        n_pages, page_size, n_kv, dim = shape
        if st[3] != 1:
            raise ValueError("the elements of a head must be adjacent")
        table_shape, table_st = page_table.shape, page_table.stride()
        if len(table_shape) != 2 or page_table.dtype is not torch.int32 or \
                (table_shape[1] > 1 and table_st[1] != 1):
            raise ValueError("page_table must be int32 [n_seq, max_pages] with adjacent columns")
        if v_pages.get_device() != index or page_table.get_device() != index:
            raise ValueError("the cache's tensors must be on one device")
        if bounds is not None and (bounds.shape != (n_pages, 2, n_kv, dim) or bounds.dtype is not dtype
                                   or not bounds.is_contiguous() or bounds.get_device() != index):
            raise ValueError("bounds must be a contiguous [n_pages, 2, n_kv_heads, head_dim] tensor "
                             "of the cache's dtype and device")
        n_seq, max_pages = table_shape
        self.k_pages, self.v_pages, self.page_table, self.bounds = k_pages, v_pages, page_table, bounds
        self.dtype, self.device, self.index, self.n_seq = dtype, k_pages.device, index, n_seq
        self.n_kv_heads, self.head_dim, self.page_size = n_kv, dim, page_size
        self.sizes = (index, n_seq, n_kv, dim, max_pages)
        # the stride of an axis of one element is never used: any valid value
        self._struct = PagedKVStruct.from_buffer_copy(_PAGED_KV.pack(
            k_pages.data_ptr(), v_pages.data_ptr(), 0 if bounds is None else bounds.data_ptr(),
            page_table.data_ptr(), st[0] if n_pages > 1 else page_size * n_kv * dim, st[1],
            st[2] if n_kv > 1 else dim, n_pages, page_size, n_kv, dim, n_seq, max_pages,
            table_st[0] if n_seq > 1 else max_pages, _DTYPES[dtype]))
        self.ref = byref(self._struct)


def _rows(name: str, x: torch.Tensor, kv: PagedKV, n_rows: int, n_heads: int) -> int:
    """Row stride of a [n_rows, n_heads, head_dim] tensor whose rows are head-contiguous."""
    dim = kv.head_dim
    if x.shape != (n_rows, n_heads, dim):
        raise ValueError(f"{name} has shape {tuple(x.shape)}: expected [{n_rows}, {n_heads}, {dim}]")
    row, head, el = x.stride()
    if x.dtype is not kv.dtype or x.get_device() != kv.index:
        raise ValueError(f"{name} must be {kv.dtype} on {kv.device}")
    if el != 1 or (head != dim and n_heads > 1):
        raise ValueError(f"{name}: the heads of a row must be adjacent")
    return row if n_rows > 1 else n_heads * dim


def _ints(name: str, x: torch.Tensor, kv: PagedKV, n: int) -> int:
    """Address of a contiguous int32 (or uint32) vector of n values."""
    if (x.dtype is not torch.int32 and x.dtype is not torch.uint32) or x.get_device() != kv.index or \
            x.shape != (n,) or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} values on {kv.device}")
    return x.data_ptr()


def _heads(q: torch.Tensor) -> int:
    if q.dim() != 3:
        raise ValueError(f"q has shape {tuple(q.shape)}: expected [rows, heads, head_dim]")
    return q.shape[1]


def _call(kv: PagedKV, fn, *args) -> None:
    """A library entry on the cache's device and its current stream (appended)."""
    index = kv.index
    if index == _current_device():
        rc = fn(kv.ref, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(kv.ref, *args, _raw_stream(index))
    if rc:
        check(rc)


def _workspace_need(kv: PagedKV, query: str, *sizes) -> int:
    """Bytes that the library function `query` asks for on the current device, remembered.
    (Not an answer of 0: other calls of the same key may differ in what was refused.)"""
    need = getattr(lib(), query)(kv.ref, *sizes)
    if need:
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        _workspace_bytes[query, sizes, kv.sizes] = need
    return need


def _workspace(kv: PagedKV, query: str, *sizes) -> tuple:
    """(memory, bytes) that the library function `query` asks for."""
    need = _workspace_bytes.get((query, sizes, kv.sizes))
    if need is None:
        with torch.cuda.device(kv.index):
            need = _workspace_need(kv, query, *sizes)
    return kv.k_pages.new_empty((need + 1) >> 1), need   # of 16-bit elements


def rope_append_paged(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      seq_len: torch.Tensor, inv_freq: torch.Tensor,
                      cu_tokens: torch.Tensor | None = None, interleaved: bool = False,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """apply_rope_q4 and write_kv_cache (rope.metal:12-39, attention.metal:67-84)
    of a batch of new tokens over a paged cache (qwen_rope_append_paged): rotates
    q [n, heads, d] into `out` (which may be q; new memory by default), writes
    rotated k and v [n, kv_heads, d] to the cache and keeps its bounds.

    seq_len [n_seq] counts the new tokens.  cu_tokens int32 [n_seq + 1]: sequence s
    owns rows cu_tokens[s]:cu_tokens[s + 1], its last positions; rows behind the last
    sequence are not touched.  None: row s is sequence s's newest token, and a
    sequence of length 0 is passed over.  inv_freq: fp32 [rot_dim / 2]."""
    heads, n = _heads(q), q.shape[0]
    qs = _rows("q", q, kv, n, heads)
    ks = _rows("k", k, kv, n, kv.n_kv_heads)
    vs = _rows("v", v, kv, n, kv.n_kv_heads)
    if out is None:
        out = q.new_empty(n, heads, kv.head_dim)
        os_ = heads * kv.head_dim
    else:
        os_ = _rows("out", out, kv, n, heads)
    if inv_freq.dtype is not torch.float32 or inv_freq.get_device() != kv.index or \
            inv_freq.dim() != 1 or not inv_freq.is_contiguous() or 2 * inv_freq.shape[0] > _UINT32:
        raise ValueError(f"inv_freq must be a contiguous float32 vector on {kv.device}")
    _call(kv, lib().qwen_rope_append_paged, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
          out.data_ptr(), os_, heads, n, _ints("seq_len", seq_len, kv, kv.n_seq),
          None if cu_tokens is None else _ints("cu_tokens", cu_tokens, kv, kv.n_seq + 1),
          inv_freq.data_ptr(), 2 * inv_freq.shape[0], 1 if interleaved else 0)
    return out


def _attend(kv, fn, query, sizes, lead, q, seq_len, extra, scale, out, return_lse):
    n, dim = kv.n_seq, kv.head_dim
    heads = _heads(q)
    qs = _rows("q", q, kv, n, heads)
    if out is None:
        out = q.new_empty(n, heads, dim)
        os_ = heads * dim
    else:
        os_ = _rows("out", out, kv, n, heads)
    lse = lp = None
    if return_lse:
        lse = torch.empty_strided((n, heads), (heads, 1), dtype=torch.float32, device=kv.device)
        lp = lse.data_ptr()
    ws, need = _workspace(kv, query, heads, *sizes)
    _call(kv, fn, *lead, q.data_ptr(), qs, out.data_ptr(), os_, lp, heads,
          _ints("seq_len", seq_len, kv, n), *extra, dim ** -0.5 if scale is None else scale,
          ws.data_ptr(), need)
    return (out, lse) if return_lse else out


def attention_paged(kv: PagedKV, q: torch.Tensor, seq_len: torch.Tensor, scale: float | None = None,
                    out: torch.Tensor | None = None, return_lse: bool = False):
    """attention_decode_batched over a paged cache (qwen_attention_paged): q
    [n_seq, heads, d] against each sequence's seq_len positions.  scale defaults to
    d ** -0.5; lse is the natural log of the sum of exp(scale q K^T), [n_seq, heads]
    fp32.  A sequence of length 0 gives zeros and -inf."""
    return _attend(kv, lib().qwen_attention_paged, "qwen_attention_paged_workspace", (), (), q, seq_len, (),
                   scale, out, return_lse)


def attention_prefix_paged(kv: PagedKV, q: torch.Tensor, seq_len: torch.Tensor,
                           prefix_pages: torch.Tensor, prefix_len: int, scale: float | None = None,
                           out: torch.Tensor | None = None, return_lse: bool = False):
    """attention_paged where every sequence begins with the same prefix_len
    positions, held once in pool pages prefix_pages (int32), read once for the batch
    (qwen_attention_prefix_paged).  seq_len and the page table describe what follows
    the prefix.  Weights are rounded once to the cache's type before the product with V
    (prefix_len > 0), attention_paged's to twice its digits."""
    pages = _ints("prefix_pages", prefix_pages, kv, prefix_pages.numel())
    if not 0 <= prefix_len <= _UINT32 or prefix_pages.numel() * kv.page_size < prefix_len:
        raise ValueError(f"prefix_len={prefix_len} in {prefix_pages.numel()} pages")
    return _attend(kv, lib().qwen_attention_prefix_paged, "qwen_attention_prefix_paged_workspace",
                   (prefix_len,), (), q, seq_len, (pages, prefix_len), scale, out, return_lse)


def select_pages(kv: PagedKV, q: torch.Tensor, seq_len: torch.Tensor, n_select: int, n_first: int = 1,
                 n_last: int = 1, out: torch.Tensor | None = None) -> torch.Tensor:
    """The n_select pages of each sequence and kv head whose bounds promise the
    highest scores for q [n_seq, heads, d] (qwen_select_pages): int32
    [n_seq, kv_heads, n_select] page-table columns, ascending, -1 behind the last.
    The first n_first and last n_last pages are always among them; ties go to the
    lower page."""
    if not (1 <= n_select <= _UINT32 and 0 <= n_first <= _UINT32 and 0 <= n_last <= _UINT32):
        raise ValueError(f"n_select={n_select} n_first={n_first} n_last={n_last}")
    heads, n = _heads(q), kv.n_seq
    qs = _rows("q", q, kv, n, heads)
    shape = (n, kv.n_kv_heads, n_select)
    if out is None:
        out = kv.page_table.new_empty(*shape)
    elif out.shape != shape or out.dtype is not torch.int32 or out.get_device() != kv.index or \
            not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int32 tensor {shape} on {kv.device}")
    ws, need = _workspace(kv, "qwen_select_pages_workspace")
    _call(kv, lib().qwen_select_pages, q.data_ptr(), qs, heads, _ints("seq_len", seq_len, kv, n), n_select,
          n_first, n_last, out.data_ptr(), ws.data_ptr(), need)
    return out


def attention_sparse_paged(kv: PagedKV, q: torch.Tensor, seq_len: torch.Tensor, pages: torch.Tensor,
                           scale: float | None = None, out: torch.Tensor | None = None,
                           return_lse: bool = False):
    """attention_paged over the listed pages alone (qwen_attention_sparse_paged):
    pages int32 [n_seq, kv_heads, n], page-table columns, -1 for none (a
    select_pages result); only positions below seq_len count."""
    n = pages.shape[-1] if pages.dim() == 3 else 0
    if pages.shape != (kv.n_seq, kv.n_kv_heads, n) or n > _UINT32 or pages.dtype is not torch.int32 or \
            pages.get_device() != kv.index or not pages.is_contiguous():
        raise ValueError(f"pages must be a contiguous int32 [{kv.n_seq}, {kv.n_kv_heads}, n] tensor "
                         f"on {kv.device}")
    return _attend(kv, lib().qwen_attention_sparse_paged, "qwen_attention_sparse_paged_workspace", (n,),
                   (pages.data_ptr(), n), q, seq_len, (), scale, out, return_lse)
