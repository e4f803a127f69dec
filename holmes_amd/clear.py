"""The cleartext model's operators that stand beside the encrypted layer.

An encrypted layer is set up from what the cleartext model does: ``DecodeSpec`` takes the shift and
the interval of the softmax's scores and the interval of their exponentials' sum from calibrated
ranges, and the decrypted answers are judged by the probabilities that they give to known tokens.  The
operators here run that model's attention over real prompts at their full length:

* ``ClearKVPages``: a key/value cache in 4 bits on the GPU, in pages of 128 tokens like the encrypted
  cache's; ``append`` quantises keys and values as they are written, ``read`` gives back what is held,
  ``attend`` is the attention of queries over it, with the log of every row's sum of exponentials and
  the least and largest of its scores;
* ``softmax_ranges``: the encrypted softmax's shift and intervals from those;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives of logits.

Values are held as a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 units.  A unit is 2^(b - 127) with one byte
b for each run of 32 values along the head dimension: b is the exponent of the run's largest magnitude
rounded to one mantissa bit, less 2 (kept in 2..252), so the largest becomes 4 or 6 units and no value is
off by more than half a step.  A run that holds an infinity or a NaN is held, and read, as NaN.

Everything runs in libholmes_ckks on the current stream without synchronising; there is no CPU path.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _native as nat

__all__ = ["PAGE_TOKENS", "Attended", "ClearKVPages", "SoftmaxRanges", "TokenScores", "softmax_ranges",
           "token_logprobs"]

PAGE_TOKENS = 128

_TYPES = {torch.bfloat16: nat.HCK_BF16, torch.float16: nat.HCK_F16, torch.float32: nat.HCK_F32}


class Attended(NamedTuple):
    """Outputs [tokens][query heads][head_dim] in the queries' type; log sum exp of the scaled scores and,
    where asked for, the least and largest of them, [tokens][query heads] float32.  A row that sees no
    token gives 0, -inf, +inf and -inf."""

    out: torch.Tensor
    lse: torch.Tensor
    low: torch.Tensor | None
    high: torch.Tensor | None


class TokenScores(NamedTuple):
    """Of every row of logits: the given token's log probability, the entropy in nats, and the ``top`` most
    likely tokens (the lower one first where they tie) with their log probabilities."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


class SoftmaxRanges(NamedTuple):
    """``DecodeSpec``'s ``score_shift``, ``exp_interval`` and ``rsqrt_interval``."""

    score_shift: float
    exp_interval: tuple
    rsqrt_interval: tuple


# A call on a few tokens costs what the host does for it: checks are one plain condition, looked at again
# one by one only where it fails, and tensors are made by the cheapest call.
def _no_type(dtype: torch.dtype, allowed, what: str):
    return ValueError(f"{what} must be {', '.join(str(d).replace('torch.', '') for d in allowed)}, not {dtype}")


_QUERY_TYPES = {torch.bfloat16: nat.HCK_BF16, torch.float16: nat.HCK_F16}
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(index) without its object
_empty = torch.empty_strided


class ClearKVPages:
    """``pages`` pages of 128 tokens for ``kv_heads`` heads, keys and values: 136 bytes a token and head of
    128 dims.  Slots are numbered page * 128 + place; which sequence holds which pages is the caller's
    table."""

    def __init__(self, pages: int, kv_heads: int = 8, head_dim: int = 128, device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if pages < 1 or not 1 <= kv_heads <= 65535:
            raise ValueError("a pool needs pages >= 1 and 1 <= kv_heads <= 65535")
        if torch.device(device).type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("cleartext pages live on a GPU: there is no CPU path")
        self.pages, self.kv_heads, self.head_dim = int(pages), int(kv_heads), int(head_dim)
        self._lib = nat.lib()
        self.buf = torch.zeros((self.pages, self.kv_heads, self._lib.hck_kv4_page_bytes(self.head_dim)),
                               dtype=torch.uint8, device=device)
        self._at, self._device, self._index = self.buf.data_ptr(), self.buf.device, self.buf.device.index

    @property
    def device(self) -> torch.device:
        return self.buf.device

    @property
    def nbytes(self) -> int:
        return int(self.buf.numel())

    def _slots(self, slots) -> torch.Tensor:
        if slots.dim() != 1 or slots.dtype != torch.int64 or slots.device != self._device:
            raise ValueError("slots must be a 1-d int64 tensor on the pool's device")
        return slots if slots.is_contiguous() else slots.contiguous()

    def append(self, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes ``keys`` and ``values`` [tokens][kv_heads][head_dim] (bf16, fp16 or fp32, any strides but
        the last axis contiguous) into ``slots`` [tokens].  A slot outside the pool, as -1 for padding, leaves
        its token out; the slots of one call must differ."""

        slots = self._slots(slots)
        tokens, device, dtype = slots.numel(), self._device, keys.dtype
        shape, kind = (tokens, self.kv_heads, self.head_dim), _TYPES.get(dtype)
        if kind is None:
            raise _no_type(dtype, _TYPES, "keys")
        if keys.shape != shape or values.shape != shape or values.dtype != dtype or keys.device != device \
                or values.device != device or keys.stride(2) != 1 or values.stride(2) != 1:
            raise ValueError(f"keys and values must be {list(shape)}, contiguous along the last axis, in one type on the "
                             "pool's device")
        k_token, k_head, _ = keys.stride()
        v_token, v_head, _ = values.stride()
        err = self._lib.hck_kv4_append(self._at, self.pages, self.kv_heads, self.head_dim, kind, keys.data_ptr(), k_token,
                                       k_head, values.data_ptr(), v_token, v_head, slots.data_ptr(), tokens,
                                       _raw_stream(self._index))
        if err:
            nat.check(err, "hck_kv4_append")

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple:
        """What ``slots`` hold, as ``(keys, values)`` [tokens][kv_heads][head_dim] in ``dtype``: exact in bf16
        and fp32; in fp16 rounded, with its largest value for any above.  Zeros for a slot outside the pool."""

        slots = self._slots(slots)
        tokens, heads, dim, kind = slots.numel(), self.kv_heads, self.head_dim, _TYPES.get(dtype)
        if kind is None:
            raise _no_type(dtype, _TYPES, "dtype")
        keys = _empty((tokens, heads, dim), (heads * dim, dim, 1), dtype=dtype, device=self._device)
        values = torch.empty_like(keys)
        err = self._lib.hck_kv4_read(self._at, self.pages, heads, dim, kind, slots.data_ptr(), tokens, keys.data_ptr(),
                                     values.data_ptr(), _raw_stream(self._index))
        if err:
            nat.check(err, "hck_kv4_read")
        return keys, values

    def attend(self, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               starts: torch.Tensor | None = None, most: int | None = None, causal: bool = True,
               scale: float | None = None, ranges: bool = False) -> Attended:
        """Attention of ``queries`` [tokens][query heads][head_dim] (bf16 or fp16, any strides but the last
        axis contiguous; query heads a multiple of kv_heads, neighbours sharing a key head) over the cache.

        Sequence b holds the pages ``table[b]`` (int32 [sequences][columns]) and ``lengths[b]`` (int32) tokens.
        Its queries are rows ``starts[b] .. starts[b + 1]`` (int32 [sequences + 1]; without ``starts`` the one
        row b), and stand for its last tokens: query i of n sees the tokens up to length - n + i, or, with
        ``causal`` off, all.  ``most`` bounds the queries of one sequence (default: 1 without ``starts``, else
        all rows) and only saves work; a sequence with more has the rest left unwritten, as has any row that no
        sequence covers.  A page outside the pool counts as tokens that are not there.  ``scale`` multiplies
        the scores (default head_dim^-1/2); ``ranges`` asks for their least and largest."""

        dim, kv_heads, dev, lib = self.head_dim, self.kv_heads, self._device, self._lib
        i32, kind = torch.int32, _QUERY_TYPES.get(queries.dtype)
        if kind is None:
            raise _no_type(queries.dtype, _QUERY_TYPES, "queries")
        if queries.dim() != 3 or queries.shape[2] != dim or queries.stride(2) != 1 or queries.device != dev:
            raise ValueError(f"queries must be [tokens][query heads][{dim}], contiguous along the last axis, on the "
                             "pool's device")
        tokens, heads, _ = queries.shape
        if heads == 0 or heads % kv_heads:
            raise ValueError(f"query heads must be a multiple of {kv_heads}")
        if table.dim() != 2 or lengths.dim() != 1 or table.shape[0] != lengths.shape[0]:
            raise ValueError("table must be [sequences][columns] and lengths [sequences]")
        seqs, cols = table.shape
        if table.dtype != i32 or lengths.dtype != i32 or table.device != dev or lengths.device != dev \
                or (table.stride(1) != 1 and table.numel()) or (lengths.stride(0) != 1 and seqs):
            raise ValueError("table and lengths must be int32 on the pool's device, contiguous along the last axis")
        if starts is None:
            if tokens != seqs:
                raise ValueError("starts must be [sequences + 1], or there is one query for each sequence")
            first, most = None, 1 if most is None else min(int(most), tokens)
        else:
            if starts.shape != (seqs + 1,):
                raise ValueError("starts must be [sequences + 1], or there is one query for each sequence")
            if starts.dtype != i32 or starts.device != dev or starts.stride(0) != 1:
                raise ValueError("starts must be int32 on the pool's device, contiguous along the last axis")
            first, most = starts.data_ptr(), tokens if most is None else min(int(most), tokens)
        if most < 0:
            raise ValueError("most must not be negative")
        scale = dim**-0.5 if scale is None else float(scale)
        if not 0.0 < scale < math.inf:
            raise ValueError("scale must be positive and finite")
        group = heads // kv_heads
        out = _empty((tokens, heads, dim), (heads * dim, dim, 1), dtype=queries.dtype, device=dev)
        low = high = low_at = high_at = None
        if ranges:
            lse, low, high = _empty((3, tokens, heads), (tokens * heads, heads, 1), dtype=torch.float32, device=dev).unbind(0)
            low_at, high_at = low.data_ptr(), high.data_ptr()
        else:
            lse = _empty((tokens, heads), (heads, 1), dtype=torch.float32, device=dev)
        need = lib.hck_kv4_attend_workspace_bytes(tokens, seqs, kv_heads, group, dim, most, cols)
        work = _empty((need,), (1,), dtype=torch.uint8, device=dev) if need else None
        err = lib.hck_kv4_attend(
            self._at, self.pages, kv_heads, dim, kind, queries.data_ptr(), tokens, group, queries.stride(0),
            queries.stride(1), table.data_ptr(), table.stride(0), cols, lengths.data_ptr(), first, seqs, most, int(causal),
            scale, out.data_ptr(), lse.data_ptr(), low_at, high_at, work.data_ptr() if need else None, need,
            _raw_stream(self._index))
        if err:
            nat.check(err, "hck_kv4_attend")
        return Attended(out, lse, low, high)


def softmax_ranges(low: torch.Tensor, high: torch.Tensor, lse: torch.Tensor, margin: float = 0.05) -> SoftmaxRanges:
    """The encrypted softmax's shift U and intervals for the rows that ``attend(..., ranges=True)`` saw:
    mapped = (s - U) / 2 runs over ``exp_interval``, made even about 0, and sum exp(2 mapped) over
    ``rsqrt_interval``, both widened by ``margin`` of their width (of their logarithm's, for the sum).  Rows
    that see no token do not count."""

    seen = torch.isfinite(lse)
    if not bool(seen.any()):
        raise ValueError("no row saw a token")
    lo, hi = float(low[seen].min()), float(high[seen].max())
    shift = 0.5 * (lo + hi)
    half = max(0.25 * (hi - lo) * (1.0 + 2.0 * margin), 1e-3)
    a, b = float(lse[seen].min()) - shift, float(lse[seen].max()) - shift
    pad = max(margin * (b - a), 1e-3)
    return SoftmaxRanges(shift, (-half, half), (math.exp(a - pad), math.exp(b + pad)))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0) -> TokenScores:
    """Scores of ``logits`` [rows][vocabulary] (bf16, fp16 or fp32, rows any distance apart) in float32: log
    probabilities of ``tokens`` [rows] int64 (a negative one, as of padding, gives 0; one past the vocabulary
    NaN), the entropies, and the ``top`` (up to 32) most likely tokens, int64 and log probabilities.  A logit
    of -inf is a token that cannot be; a row of nothing else gives -inf, and 0 for the entropy."""

    kind = _TYPES.get(logits.dtype)
    if kind is None:
        raise _no_type(logits.dtype, _TYPES, "logits")
    if logits.dim() != 2 or logits.shape[1] < 1 or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be [rows][vocabulary], contiguous along the last axis")
    rows, vocab = logits.shape
    if not 0 <= top <= min(nat.HCK_TOP_MAX, vocab):
        raise ValueError(f"top must be in 0..{min(nat.HCK_TOP_MAX, vocab)}")
    dev = logits.device
    if tokens is not None:
        if tokens.shape != (rows,) or tokens.dtype != torch.int64 or tokens.device != dev:
            raise ValueError("tokens must be [rows] int64 on the logits' device")
        tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    if dev.type != "cuda":
        raise RuntimeError("token scores run on a GPU: there is no CPU path")
    lib, f32 = nat.lib(), torch.float32
    entropy = _empty((rows,), (1,), dtype=f32, device=dev)
    given = given_at = tokens_at = ids = logs = ids_at = logs_at = None
    if tokens is not None:
        given = torch.empty_like(entropy)
        given_at, tokens_at = given.data_ptr(), tokens.data_ptr()
    if top:
        ids = _empty((rows, top), (top, 1), dtype=torch.int64, device=dev)
        logs = _empty((rows, top), (top, 1), dtype=f32, device=dev)
        ids_at, logs_at = ids.data_ptr(), logs.data_ptr()
    need = lib.hck_token_scores_workspace_bytes(rows, vocab, kind, top)
    work = _empty((need,), (1,), dtype=torch.uint8, device=dev) if need else None
    err = lib.hck_token_scores(logits.data_ptr(), kind, rows, vocab, logits.stride(0), tokens_at, top, given_at,
                               entropy.data_ptr(), ids_at, logs_at, work.data_ptr() if need else None, need,
                               _raw_stream(dev.index))
    if err:
        nat.check(err, "hck_token_scores")
    return TokenScores(given, entropy, ids, logs)
