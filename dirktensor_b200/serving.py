"""Serving operators over the C ABI: a paged K/V cache of 8-bit codes, the attention of new
tokens that reads it (alone, or behind a prefix that a batch shares), and log probabilities of
given tokens with their gradient.

Arguments are CUDA torch tensors; calls run on the current stream of the tensors' device, do not
synchronise, and raise ``ValueError`` for arguments they cannot take and ``DTError`` for
what the library refuses.  None records autograd history.  The reference has no counterpart: it recomputes every prefix, and its
CrossEntropyLoss.cpp:8-43 reduces the loss to one number.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ._lib import check, dt_kv_cache, lib
from .attention import FlashAttentionResult, head_dim, n_heads

_CODES = {"int8": (torch.int8, 0), "e4m3": (torch.float8_e4m3fn, 1)}
_FORMAT_OF = {torch.int8: 0, torch.float8_e4m3fn: 1}
_VALUES = (torch.bfloat16, torch.float32)
_INT_MAX = 2**31 - 1  # counts are ints at the C ABI


# A decoding step's calls take a few microseconds on the GPU, so the checks below look at each
# tensor as few times as they can.
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


def _call(index: int, function, *args) -> None:
    """Calls an entry point on the current stream of device `index`, which is made the current device."""
    if _current_device() == index:
        status = function(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, _current_stream(index))
    if status:
        check(status)


def _index_of(t) -> int:
    """The device of a CUDA tensor, -1 for anything else."""
    return t.get_device() if isinstance(t, torch.Tensor) else -1


def _new(shape, dtype, device):
    """torch.empty(shape), whose own checks take a microsecond more than empty_strided's."""
    strides, n = [1] * len(shape), 1
    for i in range(len(shape) - 1, -1, -1):
        strides[i] = n
        n *= shape[i] or 1
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


def _values(name: str, t, index: int, heads: Optional[int] = None):
    """Shape and strides (of sequences and tokens) of [B, T, heads, 128] of bf16 or fp32 whose rows start on 16-byte
    boundaries.  The stride of a dimension of one leads nowhere and counts as 0."""
    if _index_of(t) != index or t.dtype not in _VALUES or t.dim() != 4 or t.shape[3] != head_dim:
        raise ValueError(f"{name} must be a bfloat16 or float32 tensor [B, T, heads, {head_dim}] on cuda:{index}")
    shape, s = t.shape, t.stride()
    if shape[0] * shape[1] > _INT_MAX:  # (a broadcast tensor)
        raise ValueError(f"{name} has too many tokens")
    if heads is not None and shape[2] != heads:
        raise ValueError(f"{name} must have {heads} heads")
    batch, token = s[0] if shape[0] > 1 else 0, s[1] if shape[1] > 1 else 0
    if ((s[3] != 1 or (s[2] != head_dim and shape[2] > 1) or (batch | token) % (16 // t.element_size())
         or t.data_ptr() & 15) and t.numel()):
        raise ValueError(f"{name}: heads must be {head_dim} apart, and rows must start on 16-byte boundaries")
    return shape, (batch, token)


def _ints(name: str, t, index: int, n: Optional[int]):
    if t is None:
        return None
    if (_index_of(t) != index or t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n)
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor{'' if n is None else f' of {n} entries'} "
                         f"on cuda:{index}")
    return t.data_ptr()


def _table(t, index: int, B: int):
    if _index_of(t) != index or t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != B:
        raise ValueError(f"page_table must be an int32 tensor [{B}, pages] on cuda:{index}")
    n = t.shape[1]
    row, column = t.stride()
    if (n > 1 and column != 1) or (B > 1 and row < n):
        raise ValueError("page_table rows must be contiguous and must not overlap")
    return t.data_ptr(), max(row, n), n


class KVCache:
    """A pool of pages that holds K and V of past tokens as 8-bit codes, one fp32 scale per row of
    128 values: ``k``, ``v`` [num_pages, kv_heads, page_size, 128] (``torch.int8`` or
    ``torch.float8_e4m3fn``), ``k_scale``, ``v_scale`` [num_pages, kv_heads, page_size].

    The caller hands out pages: ``page_table`` [B, pages] (int32) names, for each sequence, the
    page of its first ``page_size`` tokens, then of the next, and so on.  Entries that no token
    reaches yet may be anything; a page id outside the pool is skipped, not followed.
    """

    def __init__(self, num_pages: int, page_size: int = 64, kv_heads: int = n_heads, format: str = "int8",
                 device: int = 0):
        if format not in _CODES:
            raise ValueError(f"format must be one of {sorted(_CODES)}")
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        shape = (int(num_pages), int(kv_heads), int(page_size))
        codes = [torch.zeros(shape + (head_dim,), dtype=torch.int8, device=dev).view(_CODES[format][0])
                 for _ in range(2)]
        self._take(*codes, *(torch.zeros(shape, dtype=torch.float32, device=dev) for _ in range(2)))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "KVCache":
        """A cache over the caller's own arrays, in the layout above.  ``append`` needs four that do not overlap."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, k_scale, v_scale):
        if not (isinstance(k, torch.Tensor) and k.is_cuda and k.dtype in _FORMAT_OF and k.dim() == 4
                and k.shape[3] == head_dim):
            raise ValueError(f"k must be an int8 or float8_e4m3fn CUDA tensor [pages, heads, page_size, {head_dim}]")
        for name, t, shape, dtype in (("k", k, k.shape, k.dtype), ("v", v, k.shape, k.dtype),
                                      ("k_scale", k_scale, k.shape[:3], torch.float32),
                                      ("v_scale", v_scale, k.shape[:3], torch.float32)):
            if not (isinstance(t, torch.Tensor) and t.device == k.device and t.dtype == dtype and t.shape == shape
                    and t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {k.device}")
        self._arrays = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size = k.shape[:3]
        if self.page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        self.device, self._index = k.device, k.get_device()
        self._c = dt_kv_cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.num_pages,
                              self.page_size, self.kv_heads, _FORMAT_OF[k.dtype])
        self._ref = ctypes.byref(self._c)

    # (the library keeps their addresses: they are not to be replaced)
    k = property(lambda self: self._arrays[0])
    v = property(lambda self: self._arrays[1])
    k_scale = property(lambda self: self._arrays[2])
    v_scale = property(lambda self: self._arrays[3])

    @property
    def format(self) -> str:
        return "int8" if self.k.dtype == torch.int8 else "e4m3"

    def append(self, k, v, page_table, start=None, lens=None) -> None:
        """Quantises k, v [B, T, kv_heads, 128] (bf16 or fp32) into the cache: token t < lens[b]
        of sequence b at position start[b] + t.  start, lens: int32 [B] tensors (default 0 and
        T).  Tokens without a valid page are skipped; where the page table gives two tokens of
        the call one slot, the one of the highest (sequence, position) is kept."""
        (B, T, _, _), ks = _values("k", k, self._index, self.kv_heads)
        _, vs = _values("v", v, self._index, self.kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v differ in shape or type")
        table, stride, n = _table(page_table, self._index, B)
        _call(self._index, lib().dt_kv_cache_append, self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              k.dtype == torch.float32, table, stride, n, _ints("start", start, self._index, B),
              _ints("lens", lens, self._index, B), B, T)

    def read(self, page_table, start, T: int, lens=None, dtype=torch.bfloat16):
        """The values of positions start[b] .. start[b] + T - 1 as k, v [B, T, kv_heads, 128] of
        ``dtype`` (bf16 or fp32).  Rows t >= lens[b] and positions without a valid page are zeros."""
        if dtype not in _VALUES:
            raise ValueError("dtype must be bfloat16 or float32")
        if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
            raise ValueError("page_table must be an int32 tensor [B, pages]")
        B, T = page_table.shape[0], int(T)
        if not 0 <= T <= _INT_MAX:
            raise ValueError("T must be >= 0 and below 2^31")
        table, stride, n = _table(page_table, self._index, B)
        k = _new((B, T, self.kv_heads, head_dim), dtype, self.device)
        v = torch.empty_like(k)
        _call(self._index, lib().dt_kv_cache_read, self._ref, k.data_ptr(), v.data_ptr(), dtype == torch.float32, table,
              stride, n, _ints("start", start, self._index, B), _ints("lens", lens, self._index, B), B, T)
        return k, v


def _outputs(q, shape, out, return_stats):
    """Output and statistics tensors, and their addresses."""
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else _new(shape, q.dtype, q.device)
    elif not (out.device == q.device and out.dtype == q.dtype and out.shape == shape and out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor of q's shape and type")
    if not return_stats:
        return out, None, None, out.data_ptr(), None, None
    m, l = (_new(shape[:3], torch.float32, q.device) for _ in range(2))
    return out, m, l, out.data_ptr(), m.data_ptr(), l.data_ptr()


_workspace_bytes: dict = {}


def _workspace(cache, *sizes):
    """A workspace of its own for each call (from torch's caching allocator, which knows streams and
    captured graphs), and its address and size."""
    nbytes = _workspace_bytes.get(sizes)
    if nbytes is None:
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        nbytes = _workspace_bytes[sizes] = (lib().dt_prefix_attn_workspace_bytes(*sizes))
    if nbytes == 0:
        return None, None, 0
    ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=cache.device)
    return ws, ws.data_ptr(), nbytes


def cache_attention_forward(q, cache: KVCache, page_table, seq_lens, scale: float, q_lens=None, out=None,
                            return_stats: bool = False):
    """Attention of new tokens over the cache; flash_attention_forward's form for single tokens.

    q: [B, T, heads, 128] bf16 or fp32, heads a multiple of the cache's.  seq_lens (int32 [B])
    counts each sequence's tokens in the cache, the queries' own included: query t sees the keys
    j < seq_lens[b] - q_lens[b] + t + 1.  q_lens (int32 [B], default T): rows past it are padding
    and come back as zeros, as do rows that see no key.  ``out`` may be a contiguous q itself, and must
    not overlap it otherwise.  Returns the output [B, T, heads, 128] of q's type, or with return_stats a ``FlashAttentionResult`` with softmax_m and softmax_l.
    """
    index = cache._index
    shape, s = _values("q", q, index)
    B, T, H, _ = shape
    table, stride, n = _table(page_table, index, B)
    lens = _ints("seq_lens", seq_lens, index, B)
    f32 = q.dtype == torch.float32
    o, m, l, po, pm, pl = _outputs(q, shape, out, return_stats)
    ws, pw, nbytes = _workspace(cache, B, T, H, cache.kv_heads, f32, cache.page_size, n, 0)
    _call(index, lib().dt_cache_attn_fwd, cache._ref, q.data_ptr(), s[0], s[1], f32, po, pm, pl, table, stride, n, lens,
          _ints("q_lens", q_lens, index, B), B, T, H, float(scale), pw, nbytes)
    return FlashAttentionResult(o, m, l) if return_stats else o


def prefix_attention_forward(q, cache: KVCache, prefix_pages, prefix_len: int, page_table, seq_lens, scale: float,
                             q_lens=None, out=None, return_stats: bool = False):
    """cache_attention_forward for a batch whose sequences share their first ``prefix_len`` tokens,
    kept once in the pages ``prefix_pages`` (int32): the prefix is read once for the whole batch.
    page_table and seq_lens describe what follows the prefix in each sequence; both may be None when
    nothing does.
    """
    index = cache._index
    shape, s = _values("q", q, index)
    B, T, H, _ = shape
    prefix_len = int(prefix_len)
    pages = _ints("prefix_pages", prefix_pages, index, None)
    if not 0 <= prefix_len <= min(1 << 30, 0 if prefix_pages is None else prefix_pages.shape[0] * cache.page_size):
        raise ValueError("prefix_len must be >= 0, within prefix_pages and at most 2^30")
    if (page_table is None) != (seq_lens is None):
        raise ValueError("page_table and seq_lens come together")
    table, stride, n = (None, 0, 0) if page_table is None else _table(page_table, index, B)
    lens = _ints("seq_lens", seq_lens, index, B)
    f32 = q.dtype == torch.float32
    o, m, l, po, pm, pl = _outputs(q, shape, out, return_stats)
    ws, pw, nbytes = _workspace(cache, B, T, H, cache.kv_heads, f32, cache.page_size, n, prefix_len)
    _call(index, lib().dt_prefix_attn_fwd, cache._ref, q.data_ptr(), s[0], s[1], f32, po, pm, pl, pages, prefix_len, table,
          stride, n, lens, _ints("q_lens", q_lens, index, B), B, T, H, float(scale), pw, nbytes)
    return FlashAttentionResult(o, m, l) if return_stats else o


class TokenLogProbs(NamedTuple):
    log_prob: object       # [...] log probability of each target (None without targets)
    entropy: object        # [...] of each row's distribution, in nats
    lse: object            # [...] log of the sum of exponentials
    top_ids: object        # [..., top] int32, most likely first (None for top = 0)
    top_log_probs: object  # [..., top]


def _rows(name, t):
    """(row count, row stride) of a tensor [..., V] whose rows are contiguous and evenly spaced."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _VALUES and t.dim() >= 1 and t.shape[-1] >= 1):
        raise ValueError(f"{name} must be a bfloat16 or float32 CUDA tensor [..., vocabulary]")
    V = t.shape[-1]
    if V > 1 << 30 or t.numel() > V * _INT_MAX:
        raise ValueError(f"{name} must have at most 2^30 entries a row and fewer than 2^31 rows")
    if t.is_contiguous():
        return (t.shape[0] if t.dim() == 2 else t.numel() // V), V
    n, ld = 1, None
    if V == 1 or t.stride(-1) == 1:
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if ld is None:
                ld = stride
            elif stride != n * ld:
                break
            n *= size
        else:
            if ld is None or ld >= V:  # (rows that share memory have a distance of zero)
                return n, V if ld is None else ld
    raise ValueError(f"{name}: rows must be contiguous and evenly spaced")


def _targets(targets, shape, device):
    if targets is None:
        return None, 0
    if not (isinstance(targets, torch.Tensor) and targets.device == device and targets.shape == shape
            and targets.dtype in (torch.int32, torch.int64) and targets.is_contiguous()):
        raise ValueError(f"targets must be a contiguous int32 or int64 tensor {list(shape)} on {device}")
    return targets.data_ptr(), int(targets.dtype == torch.int64)


def token_log_probs(logits, targets=None, top: int = 0) -> TokenLogProbs:
    """Log probabilities of given tokens, with each distribution's entropy and its ``top`` (0..32)
    most likely tokens.

    logits: [..., V] fp32 or bf16 (rows may be spaced apart); targets: int32 or int64 [...].
    A target outside 0..V-1, such as an ignored label's -100, gives 0.  Ties among the
    alternatives go to the lower id.  Logits of -inf have probability 0.  The results have no
    autograd history, also where the logits have one: token_log_probs_backward is the gradient.
    """
    n, ld = _rows("logits", logits)
    V, shape, dev = logits.shape[-1], logits.shape[:-1], logits.device
    t, t64 = _targets(targets, shape, dev)
    top = int(top)
    if not 0 <= top <= min(32, V):
        raise ValueError("top must be 0..32 and at most the vocabulary")
    lse = _new(shape, torch.float32, dev)
    ent = torch.empty_like(lse)
    lp = None if targets is None else torch.empty_like(lse)
    ids = tlp = None
    if top:
        tlp = _new(shape + (top,), torch.float32, dev)
        ids = torch.empty_like(tlp, dtype=torch.int32)
    _call(logits.get_device(), lib().dt_token_log_probs, logits.data_ptr(), logits.dtype == torch.float32, ld, n, V, t, t64, top,
          None if lp is None else lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), ids.data_ptr() if top else None,
          tlp.data_ptr() if top else None)
    return TokenLogProbs(lp, ent, lse, ids, tlp)


def token_log_probs_backward(logits, targets, lse, entropy, d_log_prob, d_entropy=None, out=None):
    """Gradient of token_log_probs with respect to the logits, of their shape and type, from its
    lse and entropy and the upstream gradients (fp32; d_log_prob or d_entropy may be None).
    ``out`` may be the logits themselves, and must not overlap them otherwise."""
    n, ld = _rows("logits", logits)
    V, shape, dev = logits.shape[-1], logits.shape[:-1], logits.device
    t, t64 = _targets(targets, shape, dev)
    if d_log_prob is not None and targets is None:
        raise ValueError("d_log_prob needs targets")
    if d_entropy is not None and entropy is None:
        raise ValueError("d_entropy needs entropy")
    for name, x in (("lse", lse), ("entropy", entropy), ("d_log_prob", d_log_prob), ("d_entropy", d_entropy)):
        if x is None and name != "lse":
            continue
        if not (isinstance(x, torch.Tensor) and x.device == dev and x.dtype == torch.float32 and x.shape == shape
                and x.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 tensor {list(shape)} on {dev}")
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else _new(logits.shape, logits.dtype, dev)
    elif out.device != dev or out.dtype != logits.dtype or out.shape != logits.shape:
        raise ValueError("out must have the logits' shape and type")
    dn, dld = _rows("out", out)
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    _call(logits.get_device(), lib().dt_token_log_probs_bwd, logits.data_ptr(), logits.dtype == torch.float32, ld, n, V, t,
          t64, lse.data_ptr(), ptr(entropy), ptr(d_log_prob), ptr(d_entropy), out.data_ptr(), dld)
    return out
