"""Operators of answer decoding: an 8-bit key / value cache, the attention that reads it, and beam search's two steps.

The eval loop of ``T2S`` (pythia/models/t2s.py:315-354) decodes 12 tokens against one long prefix [question; frames; OCR].  ``T2S.set_decoding``
runs it on these operators (t2s.py ``_beam_decode``); they are also usable on their own:

    cache = KVCache8(batch, heads, capacity, fmt="int8")                 # one layer
    cache.append(k, v, counts=keys.cnt, rows=keys.idx)                   # the visible rows of the prefix
    out, lse = attend(q, cache, tail_k, tail_v, tail_len)                # a few query rows, each with its own decoded tokens in the tail
    scores, parents, tokens = beam_select(logits, scores, n_beams, finished, pad)
    beam_reorder(tail, parents, batch_dim=1)

Thin wrappers over the C ABI (``include/t2s_hip.h``; kernels in ``csrc/kv8.hip`` and ``csrc/beam.hip``): shapes, types, strides and devices are
checked on the host, everything runs on the current stream of the tensors' device, without a synchronisation and without state other than
the cache's own tensors - a step may be captured into a graph.  No gradients: the operands may not require any."""
import functools
import math

import torch

from . import hipext as X

BLOCK = 64                  # tokens of a block: one scale for its keys and one for its values per head
HEAD_DIM = 64
BEAM_MAX = X.T2S_BEAM_MAX   # beams, and candidates a selection returns
FORMATS = {"int8": (X.T2S_KV_INT8, torch.int8), "e4m3": (X.T2S_KV_E4M3, torch.float8_e4m3fn)}
_empty = torch.empty_strided         # (of torch's ways to allocate the one with the least overhead: it counts in calls that take a few microseconds)
_DTYPES = {torch.float32: (X.T2S_F32, 15), torch.bfloat16: (X.T2S_BF16, 7)}          # code, mask of a 4-element alignment in bytes


def _need(ok, msg, *args):
    if not ok:
        raise ValueError(msg % args if args else msg)


def _same_device(index, *tensors):
    """All of ``tensors`` (None: absent) on GPU ``index`` and without gradients."""
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0 or t.requires_grad):
            if index < 0 or t.get_device() < 0:
                _need(index < 0, "tensors on %s and cuda:%d: all of a call's tensors live on one device", t.device, index)
                raise RuntimeError("T2S HIP kernels need device tensors (got a %s tensor); there is no CPU path" % t.device)
            _need(t.get_device() == index, "tensors on %s and cuda:%d: all of a call's tensors live on one device", t.device, index)
            _need(not torch.is_grad_enabled(), "the decode operators have no gradients: call them under torch.no_grad() or on detached tensors")


def _launch(index, fn, *args):
    """fn(*args, stream) on the current stream of GPU ``index``."""
    if index == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


# What follows from shapes, strides and types alone is checked and worked out once for each (calls of a few microseconds would spend as much on it).
def _head_strides(shape, stride, dtype, name):
    """Strides of [..., heads, 64] with dense 64-element rows that start at multiples of 4 elements (0 for axes of length 1)."""
    _need(dtype in _DTYPES, "%s: float32 or bfloat16, got %s", name, dtype)
    _need(shape[-1] == HEAD_DIM, "%s: the kernels are built for head_dim 64, got %s", name, tuple(shape))
    s = tuple(x if n > 1 else 0 for x, n in zip(stride[:-1], shape[:-1]))
    _need(stride[-1] == 1 and not any(x & 3 for x in s), "%s: rows of 64 dense elements, aligned to 4 elements, are needed (strides %s): call .contiguous()", name, stride)
    return s


def _aligned(name, mask, *addresses):
    for at in addresses:
        _need(not at & mask, "%s: rows of 64 dense elements, aligned to 4 elements, are needed (address %#x): call .contiguous()", name, at)


@functools.lru_cache(maxsize=256)
def _append_layout(B, H, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype):
    """(strides of k, strides of v, type code, alignment mask) of an append of [B, R, H, 64] rows."""
    _need(len(k_shape) == 4 and k_shape[0] == B and k_shape[2] == H and v_shape == k_shape and v_dtype == k_dtype,
          "append: k and v [%d, R, %d, 64] of one type, got %s %s and %s %s", B, H, tuple(k_shape), k_dtype, tuple(v_shape), v_dtype)
    return (_head_strides(k_shape, k_stride, k_dtype, "append: k"), _head_strides(v_shape, v_stride, v_dtype, "append: v"), *_DTYPES[k_dtype])


@functools.lru_cache(maxsize=1024)
def _attend_layout(B, H, tokens, q_shape, q_stride, q_dtype, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype):
    """Of an attention over about ``tokens`` cached tokens: the strides of q and of the tails, type code, alignment mask, shapes and strides of the
    results, shares of the token axis, bytes of workspace."""
    _need(len(q_shape) == 4 and q_shape[0] == B and q_shape[2] > 0 and q_shape[2] % H == 0, "attend: q [%d, N, a multiple of %d, 64], got %s", B, H, tuple(q_shape))
    sq, st, N, HQ = _head_strides(q_shape, q_stride, q_dtype, "attend: q"), (0, 0, 0, 0), q_shape[1], q_shape[2]
    if k_shape is not None:
        _need(len(k_shape) == 5 and k_shape == (B, N, k_shape[2], H, HEAD_DIM) and v_shape == k_shape and k_dtype == q_dtype and v_dtype == q_dtype,
              "attend: tails [%d, %d, T, %d, 64] of q's type, got %s %s and %s %s", B, N, H, tuple(k_shape), k_dtype, tuple(v_shape), v_dtype)
        st = _head_strides(k_shape, k_stride, k_dtype, "attend: tail_k")
        _need(_head_strides(v_shape, v_stride, v_dtype, "attend: tail_v") == st, "attend: tail_k and tail_v need the same strides, got %s and %s", k_stride, v_stride)
    code, mask = _DTYPES[q_dtype]
    splits, nbytes = 1, 0
    if N:
        splits = X.lib().t2s_kv8_attn_splits(B, N, H, HQ // H, tokens, code)
        nbytes = X.lib().t2s_kv8_attn_workspace_bytes(B, N, H, HQ // H, splits)
    n = HQ * HEAD_DIM
    return sq, st, code, mask, tuple(q_shape), (N * n, n, HEAD_DIM, 1), (B, N, HQ), (N * HQ, HQ, 1), splits, nbytes


@functools.lru_cache(maxsize=256)
def _select_layout(shape, stride, dtype, scores_shape, scores_dtype, finished_shape, finished_dtype, K, pad):
    """(type code, bytes of workspace) of a selection."""
    _need(len(shape) == 3 and shape[2] > 0 and shape[1] > 0, "beam_select: logits [B, N, V], got %s", tuple(shape))
    B, N, V = shape
    _need(dtype in _DTYPES, "beam_select: float32 or bfloat16 logits, got %s", dtype)
    _need(V == 1 or stride[2] == 1, "beam_select: dense rows of logits are needed (strides %s): call .contiguous()", stride)
    _need(scores_shape == (B, N) and scores_dtype == torch.float32, "beam_select: scores is float32 [%d, %d], got %s %s", B, N, tuple(scores_shape), scores_dtype)
    _need(N <= BEAM_MAX and 0 < K <= BEAM_MAX and K <= N * V, "beam_select: %d of %d x %d candidates (at most %d beams and %d candidates)", K, N, V, BEAM_MAX, BEAM_MAX)
    _need(0 <= pad < V, "beam_select: pad %d outside the vocabulary of %d", pad, V)
    _need(finished_shape is None or (finished_shape == (B, N) and finished_dtype in (torch.bool, torch.uint8)), "beam_select: finished is bool [%d, %d], got %s %s", B, N, finished_shape, finished_dtype)
    return _DTYPES[dtype][0], X.lib().t2s_beam_select_workspace_bytes(B, N, V, K)


class KVCache8:
    """Keys and values of ``batch`` sequences, ``heads`` heads of 64 dims and up to ``capacity`` tokens (rounded up to blocks of 64) in 8 bits.

    ``fmt``: "int8" (an even grid of 127 steps up to the block's largest magnitude: the finer one for projections without outliers) or "e4m3"
    (floating point, 3 fraction bits: keeps small values next to large ones).  One fp32 scale for each block of 64 tokens and head, keys and
    values apart; the storage layout is part of the C ABI (``t2s_kv8_append`` in include/t2s_hip.h).  ``k``, ``v`` [B, H, blocks, 64, 64]
    codes, ``k_scale``, ``v_scale`` [B, H, blocks], ``lens`` [B] int32: the tokens each sequence holds.

    The cache is one object of the stream's order: two appends at a time, or an append while another stream reads, are the caller's race."""

    def __init__(self, batch, heads, capacity, fmt="int8", device="cuda"):
        _need(fmt in FORMATS, "KVCache8: unknown format %r (int8 or e4m3)", fmt)
        _need(batch > 0 and heads > 0 and capacity > 0, "KVCache8: bad shape batch=%d heads=%d capacity=%d", batch, heads, capacity)
        n = -(-int(capacity) // BLOCK)
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        code = FORMATS[fmt][1]
        # (codes are written whole blocks at a time and read only below a sequence's length: nothing has to be cleared)
        k, v = (torch.empty(batch, heads, n, BLOCK, HEAD_DIM, dtype=torch.uint8, device=dev).view(code) for _ in range(2))
        ks, vs = (torch.zeros(batch, heads, n, dtype=torch.float32, device=dev) for _ in range(2))
        self._adopt(k, v, ks, vs, torch.zeros(batch, dtype=torch.int32, device=dev), 0)

    @classmethod
    def from_parts(cls, k, v, k_scale, v_scale, lens, max_len=None):
        """A cache around existing storage (used as it is, not copied): codes int8 or float8_e4m3fn [B, H, blocks, 64, 64], scales
        (positive, or NaN for a block that holds a value that is none), lens.
        ``max_len``: a bound on the lengths, if known; it only shapes the attention's launch."""
        self = cls.__new__(cls)
        self._adopt(k, v, k_scale, v_scale, lens, max_len)
        return self

    def _adopt(self, k, v, ks, vs, lens, max_len):
        fmt = [f for f, (_, t) in FORMATS.items() if t == k.dtype]
        _need(fmt and v.dtype == k.dtype, "KVCache8: codes are int8 or float8_e4m3fn, got %s and %s", k.dtype, v.dtype)
        _need(k.dim() == 5 and k.shape[3:] == (BLOCK, HEAD_DIM) and v.shape == k.shape and k.numel() > 0, "KVCache8: codes [B, H, blocks, 64, 64], got %s and %s", tuple(k.shape), tuple(v.shape))
        B, H, n = k.shape[:3]
        _need(ks.shape == (B, H, n) and vs.shape == (B, H, n) and ks.dtype == vs.dtype == torch.float32, "KVCache8: scales are float32 [B, H, blocks]")
        _need(lens.shape == (B,) and lens.dtype == torch.int32, "KVCache8: lens is int32 [B]")
        for t in (k, v, ks, vs, lens):
            _need(t.is_contiguous(), "KVCache8: the storage has to be contiguous")
            _need(t.device == k.device, "KVCache8: the storage has to live on one device")
        self.fmt, self._fmt = fmt[0], FORMATS[fmt[0]][0]
        self._parts = (k, v, ks, vs, lens)
        self.batch, self.heads, self.blocks, self.capacity, self.device = B, H, n, n * BLOCK, k.device
        self.max_len = self.capacity if max_len is None else max(0, min(int(max_len), self.capacity))
        self._ticket = torch.zeros(B, dtype=torch.int32, device=k.device)
        self._index = k.get_device()
        self._ptrs, self._ticket_ptr = tuple(t.data_ptr() for t in self._parts), self._ticket.data_ptr()

    # (the storage is fixed for the cache's life: its addresses are taken once)
    k, v, k_scale, v_scale, lens = (property(lambda self, i=i: self._parts[i]) for i in range(5))

    def __reduce__(self):
        """Copies and pickles are caches of their own storage (``copy.copy``: another handle on the same)."""
        return KVCache8.from_parts, (*self._parts, self.max_len)

    def append(self, k, v, counts=None, rows=None):
        """Puts new tokens behind what each sequence holds.  k, v: [B, R, H, 64] float32 or bfloat16, dense 64-element rows (slices of a fused
        projection are fine).  ``rows`` int32 [B, T]: token j of sequence b is row rows[b, j] of them (T = R and row j without it; an
        ``ops.KeyList``'s ``idx`` fits); ``counts`` int32 [B]: how many of the T tokens are appended (all, without it; more than T counts as T,
        less than 0 as 0).  Returns self.

        A block that holds tokens already keeps the larger of its scale and the new tokens' one; its codes are rounded again where it grew.
        A value that is not finite, or a row number outside 0 .. R - 1, turns its block of that head to NaN.  Tokens that do not fit turn the
        sequence's length to -1 and every result over it to NaN, until ``set_lens`` (the lengths live on the device: nothing is waited for)."""
        B, H = self.batch, self.heads
        sk, sv, code, mask = _append_layout(B, H, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype)
        R = T = k.shape[1]
        rp, rs, cp = None, 0, None
        if rows is not None:
            _need(rows.dim() == 2 and rows.shape[0] == B and rows.dtype == torch.int32 and (rows.shape[1] < 2 or rows.stride(1) == 1),
                  "append: rows is int32 [%d, T] with dense rows, got %s %s", B, tuple(rows.shape), rows.dtype)
            T, rp, rs = rows.shape[1], rows.data_ptr(), rows.stride(0)
        if counts is not None:
            _need(counts.shape == (B,) and counts.dtype == torch.int32 and (B == 1 or counts.stride(0) == 1), "append: counts is a dense int32 [%d]", B)
            cp = counts.data_ptr()
        elif T > self.capacity:
            _need(False, "append: %d tokens do not fit a capacity of %d", T, self.capacity)
        _need(R > 0 or T == 0, "append: %d tokens of no rows", T)
        _same_device(self._index, k, v, counts, rows)
        if T == 0:
            return self
        kp, vp = k.data_ptr(), v.data_ptr()
        if (kp | vp) & mask:
            _aligned("append", mask, kp, vp)
        X.check(_launch(self._index, X.lib().t2s_kv8_append, kp, sk[0], sk[1], sk[2], vp, sv[0], sv[1], sv[2], rp, rs, cp, *self._ptrs,
                        self._ticket_ptr, B, H, T, R, self.blocks, code, self._fmt), "t2s_kv8_append")
        self.max_len = min(self.capacity, self.max_len + T)
        return self

    def set_lens(self, lens, max_len=None):
        """Sets how many tokens each sequence holds: an int for all, or int32 [B] on the device.  Takes tokens back (a prefix is kept for another
        continuation; 0 empties the cache); it cannot bring any in, and never more may be named than have been appended.  A block that is kept in part keeps
        its scale.  ``max_len`` as in ``from_parts``."""
        if isinstance(lens, int):
            _need(0 <= lens <= self.capacity, "set_lens: %d outside 0 .. %d", lens, self.capacity)
            self.lens.fill_(lens)
            self.max_len = lens
        else:
            _need(lens.shape == (self.batch,) and lens.dtype == torch.int32, "set_lens: an int or int32 [%d], got %s %s", self.batch, tuple(lens.shape), lens.dtype)
            self.lens.copy_(lens)
        if max_len is not None:
            self.max_len = max(0, min(int(max_len), self.capacity))
        return self

    def dequantize(self, dtype=torch.bfloat16):
        """(keys, values) [B, H, capacity, 64] in ``dtype`` (float32 or bfloat16): code * scale, zeros behind a sequence's length."""
        _need(dtype in (torch.bfloat16, torch.float32), "dequantize: float32 or bfloat16, got %s", dtype)
        _same_device(self._index, self.k)
        shape, n = (self.batch, self.heads, self.capacity, HEAD_DIM), self.capacity * HEAD_DIM
        strides = (self.heads * n, n, HEAD_DIM, 1)
        k, v = _empty(shape, strides, dtype=dtype, device=self.device), _empty(shape, strides, dtype=dtype, device=self.device)
        X.check(_launch(self._index, X.lib().t2s_kv8_dequantize, *self._ptrs, k.data_ptr(), v.data_ptr(), self.batch, self.heads, self.blocks,
                        _DTYPES[dtype][0], self._fmt), "t2s_kv8_dequantize")
        return k, v


def attend(q, cache, tail_k=None, tail_v=None, tail_len=None, scale=0.125):
    """softmax(scale q k^T) v of a few query rows per sequence over what ``cache`` holds, then over each row's own tail.

    q: [B, N, HQ, 64] float32 or bfloat16 (dense 64-element rows); HQ a multiple of the cache's heads: query head i reads key head
    i // (HQ / heads).  tail_k, tail_v: [B, N, T, heads, 64] in q's type, the same strides (0 strides are fine: rows of one sequence may share
    a tail), tokens that are in no cache - a beam's decoded steps, up to a few hundred; ``tail_len``: how many of the T each row sees, int or int32
    [B, N] (all, without it; below 0 counts as 0, above T as T).  Returns (out [B, N, HQ, 64] in q's type, lse [B, N, HQ] float32: the natural
    log-sum-exp of the scaled scores).  A row that sees no token at all: out 0, lse -inf.

    Codes enter the matrix pipe exactly; a query in float32 as the three bf16 terms that make it up; probabilities in 11 bits for a bfloat16
    result (which is rounded to 8), as three bf16 terms for a float32 one.  All sums, maxima and scales are float32; the result is rounded once."""
    B, H, tokens = cache.batch, cache.heads, (cache.max_len + BLOCK - 1) // BLOCK * BLOCK
    T, tk, tv, tl, tls, layout = 0, None, None, None, (0, 0), None
    if tail_k is not None and tail_v is not None:
        layout = _attend_layout(B, H, tokens, q.shape, q.stride(), q.dtype, tail_k.shape, tail_k.stride(), tail_k.dtype, tail_v.shape, tail_v.stride(), tail_v.dtype)
        T = tail_k.shape[2]
        if torch.is_tensor(tail_len):
            _need(tail_len.shape == layout[6][:2] and tail_len.dtype == torch.int32, "attend: tail_len is an int or int32 %s", layout[6][:2])
            tl, tls = tail_len.data_ptr(), tail_len.stride()
        elif tail_len is not None:
            T = max(0, min(int(tail_len), T))
        if T > 0:
            tk, tv = tail_k.data_ptr(), tail_v.data_ptr()
    else:
        _need(tail_k is None and tail_v is None, "attend: tail_k and tail_v come together")
        _need(tail_len is None, "attend: tail_len without a tail")
        layout = _attend_layout(B, H, tokens, q.shape, q.stride(), q.dtype, None, None, None, None, None, None)
    sq, st, code, mask, shape, stride, lse_shape, lse_stride, splits, nbytes = layout
    qp = q.data_ptr()
    if (qp | (tk or 0) | (tv or 0)) & mask:
        _aligned("attend", mask, qp, tk or 0, tv or 0)
    _same_device(cache._index, q, tail_k, tail_v, None if tl is None else tail_len)
    dev = q.device
    out = _empty(shape, stride, dtype=q.dtype, device=dev)
    lse = _empty(lse_shape, lse_stride, dtype=torch.float32, device=dev)
    N, HQ = shape[1], shape[2]
    if N == 0:
        return out, lse
    ws = _empty((nbytes // 4,), (1,), dtype=torch.float32, device=dev) if nbytes else None
    X.check(_launch(cache._index, X.lib().t2s_kv8_attn, qp, sq[0], sq[1], sq[2], *cache._ptrs, tk, tv, st[0], st[1], st[2], st[3], tl, tls[0], tls[1], T,
                    out.data_ptr(), lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, splits, B, N, H, HQ // H, cache.blocks, scale, code, cache._fmt), "t2s_kv8_attn")
    return out, lse


def beam_select(logits, scores, n_select, finished=None, pad=0):
    """The ``n_select`` best continuations of each sequence's beams.

    logits [B, N, V] float32 or bfloat16 (dense rows), scores [B, N] float32: the beams' summed log-probabilities (-inf: no beam; the first step
    starts from one beam at 0 and the others at -inf).  A candidate (n, v) scores scores[b, n] + logits[b, n, v] - logsumexp(logits[b, n]).
    ``finished`` bool [B, N]: a beam that has ended offers the token ``pad`` at its own score and nothing else.  NaN logits count as -inf, +inf as
    the largest number.  Returns (scores [B, n_select] float32, parents int64: the beam n, tokens int64: the word v), best first by scores compared in 64 bits, ties
    to the lowest n V + v; candidates at -inf only where nothing else is left.  A row's logsumexp has fp32's accuracy (off by 160 2^-24 = 1e-5 at most) and
    depends on the row's logits and the call's shape, not on an address or other rows: beams of equal logits and scores tie, candidates of other beams that are closer than
    that come in either order.  At most 32 beams and 32 candidates."""
    K, pad, fp = int(n_select), int(pad), None
    if finished is None:
        code, nbytes = _select_layout(logits.shape, logits.stride(), logits.dtype, scores.shape, scores.dtype, None, None, K, pad)
    else:
        code, nbytes = _select_layout(logits.shape, logits.stride(), logits.dtype, scores.shape, scores.dtype, finished.shape, finished.dtype, K, pad)
        finished = finished.contiguous()
        fp = finished.data_ptr()
    B, N, V = logits.shape
    index = logits.get_device()
    _same_device(index, logits, scores, finished)
    dev = logits.device
    out = _empty((B, K), (K, 1), dtype=torch.float32, device=dev)
    parents, tokens = _empty((B, K), (K, 1), dtype=torch.int64, device=dev), _empty((B, K), (K, 1), dtype=torch.int64, device=dev)
    if B == 0:
        return out, parents, tokens
    scores = scores.contiguous()
    ws = _empty(((nbytes + 7) // 8,), (1,), dtype=torch.int64, device=dev) if nbytes else None
    sb, sn = logits.stride()[:2]
    X.check(_launch(index, X.lib().t2s_beam_select, logits.data_ptr(), sb, sn, scores.data_ptr(), fp, pad, out.data_ptr(), parents.data_ptr(),
                    tokens.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, B, N, V, K, code), "t2s_beam_select")
    return out, parents, tokens


def beam_reorder(state, parents, batch_dim=0, used=None):
    """state[.., b, n, ..] = state[.., b, parents[b, n], ..] in place, for every beam at once; returns ``state``.

    state: contiguous, any type; its axes ``batch_dim`` and ``batch_dim + 1`` are the sequences and their beams.  parents int64 [B, N]: any beam any
    number of times (outside 0 .. N - 1 counts as the nearest).  ``used``: only the first ``used`` entries of the axis behind the beams are moved
    (the steps decoded so far); the rest is left as it is.  At most 32 beams."""
    d = batch_dim + state.dim() if batch_dim < 0 else batch_dim
    _need(0 <= d and d + 2 <= state.dim(), "beam_reorder: batch_dim %d of a %d-d state", batch_dim, state.dim())
    B, N = state.shape[d], state.shape[d + 1]
    _need(state.is_contiguous(), "beam_reorder: the state has to be contiguous (strides %s)", state.stride())
    _need(N <= BEAM_MAX, "beam_reorder: at most %d beams, got %d", BEAM_MAX, N)
    _need(parents.shape == (B, N) and parents.dtype == torch.int64, "beam_reorder: parents is int64 [%d, %d], got %s %s", B, N, tuple(parents.shape), parents.dtype)
    rest = state.shape[d + 2:]
    row = state.element_size() * math.prod(rest)
    nbytes = row
    if used is not None:
        _need(len(rest) > 0 and 0 <= used <= rest[0], "beam_reorder: used %s of %s", used, tuple(rest))
        nbytes = row // max(1, rest[0]) * int(used)
    outer = math.prod(state.shape[:d])
    index = state.get_device()
    _same_device(index, state, parents)
    if nbytes and outer and B and N > 1:
        parents = parents.contiguous()
        X.check(_launch(index, X.lib().t2s_beam_reorder, state.data_ptr(), parents.data_ptr(), outer, B, N, row, nbytes), "t2s_beam_reorder")
    return state
