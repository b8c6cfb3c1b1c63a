"""Operators of an autoregressive text decoder over the C-ABI
(include/ppocr_b200_decode.h): a paged key/value cache held in 4 bits, the
attention that reads it, and token sampling.

torch provides device memory and streams; every call is asynchronous on the
current stream of the tensors' device. Arguments are checked here and again
at the C boundary (capi.NativeError).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import capi

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _call(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) on the device's current stream."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return capi.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    capi.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def _require(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class KvCache4:
    """A pool of pages holding keys and values in 4 bits, with a 16-bit scale
    and minimum per token, head and 32 channels (5 bits a value).

    The pool has no notion of sequences: page tables [batch, width] (int32)
    say which page holds which positions, `lengths` [batch] (int32) how many
    tokens a sequence has with the new ones, which are its last. The new
    tokens of all sequences are packed in rows; `starts` [batch + 1] (int32)
    says whose rows are whose, None that every sequence has the same number.
    `max_new` bounds the new tokens of one sequence (a host number; with
    `starts` None it follows from the row count).

    One instance serves one stream at a time: its workspace belongs to the
    attention call that is running.
    """

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cuda:0",
                 pool: torch.Tensor | None = None):
        _require(dtype in (torch.float16, torch.bfloat16), "dtype must be float16 or bfloat16")
        self.lib = capi.load()
        block = self.lib.ppocr_b200_kv4_block_bytes(page_size, head_dim)
        _require(block > 0, "page_size must be 16, 32, 64 or 128 and head_dim 32, 64 or 128")
        _require(pages > 0 and kv_heads > 0, "pages and kv_heads must be positive")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.dtype = pages, page_size, kv_heads, head_dim, dtype
        shape = (pages, kv_heads, block)
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        _require(pool.dtype == torch.uint8 and tuple(pool.shape) == shape and pool.is_contiguous()
                 and pool.device == self.device, f"pool must be a contiguous uint8 tensor {shape} on {self.device}")
        self.pool = pool
        self.workspace = torch.zeros(self.lib.ppocr_b200_kv4_workspace_bytes(), dtype=torch.uint8, device=self.device)
        self._cache = capi.PpocrKv4Cache(pool.data_ptr(), pages, page_size, kv_heads, head_dim, TYPES[dtype])
        self._ref = ctypes.byref(self._cache)

    def _places(self, table, lengths, starts, tokens: int, max_new: int | None):
        """The C-ABI's (table, width, lengths, starts, batch, tokens, max_new)."""
        dev, i32 = self.device, torch.int32
        _require(table.dtype == i32 and table.dim() == 2 and table.is_contiguous() and table.device == dev,
                 "table must be a contiguous int32 [batch, width] on the cache's device")
        batch = table.shape[0]
        _require(lengths.dtype == i32 and lengths.shape == (batch,) and lengths.is_contiguous()
                 and lengths.device == dev, "lengths must be a contiguous int32 [batch]")
        if starts is None:
            _require(tokens == 0 if batch == 0 else tokens % batch == 0,
                     "without starts, rows must divide by the batch")
            each = tokens // batch if batch else 0
            _require(max_new is None or max_new == each, "without starts, max_new is rows / batch")
            return table.data_ptr(), table.shape[1], lengths.data_ptr(), None, batch, tokens, each
        _require(starts.dtype == i32 and starts.shape == (batch + 1,) and starts.is_contiguous()
                 and starts.device == dev, "starts must be a contiguous int32 [batch + 1]")
        _require(max_new is not None, "starts needs max_new")
        return table.data_ptr(), table.shape[1], lengths.data_ptr(), starts.data_ptr(), batch, tokens, max_new

    def _rows(self, x: torch.Tensor, heads: int, what: str) -> int:
        """Row stride (elements) of [tokens, heads, head_dim] with adjacent heads."""
        d = self.head_dim
        _require(x.dtype == self.dtype and x.device == self.device and x.dim() == 3 and x.shape[1] == heads
                 and x.shape[2] == d, f"{what} must be {self.dtype} [tokens, {heads}, {d}] on {self.device}")
        s = x.stride()
        _require(s[2] == 1 and (s[1] == d or heads == 1), f"{what}'s heads must lie side by side")
        return s[0] if x.shape[0] > 1 else heads * d

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               starts: torch.Tensor | None = None, max_new: int | None = None) -> None:
        """Quantises k and v [tokens, kv_heads, head_dim] (rows may be strided)
        into the cache as each sequence's last tokens."""
        ks, vs = self._rows(k, self.kv_heads, "k"), self._rows(v, self.kv_heads, "v")
        _require(k.shape[0] == v.shape[0], "k and v must have the same rows")
        _call(self.lib.ppocr_b200_kv4_append, self.device, self._ref, k.data_ptr(), ks, v.data_ptr(), vs,
              *self._places(table, lengths, starts, k.shape[0], max_new))

    def read(self, table: torch.Tensor, lengths: torch.Tensor, tokens: int,
             starts: torch.Tensor | None = None, max_new: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [tokens, kv_heads, head_dim] that the cache holds
        for each sequence's last tokens."""
        shape = (tokens, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        _call(self.lib.ppocr_b200_kv4_read, self.device, self._ref, k.data_ptr(), v.data_ptr(),
              *self._places(table, lengths, starts, tokens, max_new))
        return k, v

    def attention(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                  starts: torch.Tensor | None = None, max_new: int | None = None, scale: float | None = None,
                  window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q [tokens, heads, head_dim] (rows may be
        strided) over the cache, which holds the tokens' own keys and values
        already. window > 0 hides positions more than window - 1 back, but for
        the first `sinks`. scale defaults to head_dim ** -0.5."""
        _require(q.dim() == 3, "q must be [tokens, heads, head_dim]")
        heads = q.shape[1]
        stride = self._rows(q, heads, "q")
        if out is None:
            out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
        else:
            _require(out.shape == q.shape and out.dtype == self.dtype and out.is_contiguous()
                     and out.device == self.device, "out must be contiguous, of q's shape, type and device")
        _call(self.lib.ppocr_b200_kv4_attention, self.device, self._ref, q.data_ptr(), stride, out.data_ptr(), heads,
              1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, sinks,
              *self._places(table, lengths, starts, q.shape[0], max_new), self.workspace.data_ptr())
        return out


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
           min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One token per row of logits [rows, vocab] (float16, bfloat16 or
    float32; rows may be strided): (ids int32, probabilities float32, numbers
    of tokens that stayed int32), each [rows]. The parameters are per row
    ([rows], float32; top_k int32), None for off; uniform [rows] float32 in
    [0, 1) decides. See include/ppocr_b200_decode.h."""
    _require(logits.dim() == 2 and logits.dtype in TYPES and logits.is_cuda and logits.stride(1) == 1,
             "logits must be a CUDA float16, bfloat16 or float32 [rows, vocab]")
    rows, vocab = logits.shape
    dev = logits.device
    ptrs = []
    for name, x, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                           ("uniform", uniform, torch.float32)):
        if x is None and name != "uniform":
            ptrs.append(None)
            continue
        _require(x is not None and x.dtype == dtype and x.shape == (rows,) and x.is_contiguous() and x.device == dev,
                 f"{name} must be a contiguous {dtype} [rows] on the logits' device")
        ptrs.append(x.data_ptr())
    ids = torch.empty(rows, dtype=torch.int32, device=dev)
    prob = torch.empty(rows, dtype=torch.float32, device=dev)
    kept = torch.empty(rows, dtype=torch.int32, device=dev)
    stride = logits.stride(0) if rows > 1 else vocab
    _call(capi.load().ppocr_b200_sample, dev, logits.data_ptr(), TYPES[logits.dtype], stride, rows, vocab, *ptrs,
          ids.data_ptr(), prob.data_ptr(), kept.data_ptr())
    return ids, prob, kept
