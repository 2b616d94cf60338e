"""What the decode operators (vitxt_gqa_amd/decode.py) are measured on.

Four operators of answer decoding against a long multimodal prefix: the 8-bit key / value cache's ``append`` (with the read-back that shows
what it holds), the attention that reads the cache (``attend``), the selection over beams and vocabulary (``beam_select``) and the
reordering of the beams' states (``beam_reorder``).  ``run`` computes each in plain torch operations, or - where ``own`` is true - through
the framework's entry points.

The cache, as a definition.  Token t of a sequence lies in block t // 64; a block of one head has one fp32 scale s for its keys and one for
its values.  Of the block's largest magnitude amax (at least 2^-100), s = amax / 127 for int8, and the least power of two with
amax <= 448 s for e4m3.  An element x is held as the int8 or e4m3 number nearest to x * r, r = 1 / s rounded to fp32, ties to even, the
product taken exactly; it stands for code * s.  An append into a block that holds tokens already keeps the larger of the old scale and
that of the new tokens, and rounds the old codes again where the scale grew.
"""
import math

import torch

own = False

BLOCK, HD = 64, 64
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}
TINY = 2.0 ** -100
# storage order of the tokens of a block in the value tensor: position p of a 64-byte row holds token ORDER[p]
ORDER = [((p >> 2) & 3) * 16 + (p >> 4) * 4 + (p & 3) for p in range(BLOCK)]


def listed():
    return [
        # the cache is filled: one newly decoded token for each of 48 answers (the repository's training batch size) behind a question of
        # up to 20 tokens and 64 frames
        dict(name="append-step", op="append", batch=48, heads=12, cap=128, new=1, held=84, fmt="int8", dtype="bf16", fused=False, listed_rows=False, seed=1),
        # the prefix of 64 questions over 100 frames x 100 OCR slots (L = 10 120), straight from the fused [B, L, 2304] projection,
        # only the rows that the mask leaves visible
        dict(name="append-prefix", op="append", batch=64, heads=12, cap=10176, new=10120, held=0, fmt="e4m3", dtype="bf16", fused=True, listed_rows=True, seed=2),
        # a ragged continuation in fp32 (the parity mode): odd counts that begin and end inside blocks
        dict(name="append-ragged", op="append", batch=7, heads=3, cap=1600, new=531, held=1001, fmt="int8", dtype="fp32", fused=False, listed_rows=False, seed=3),
        # attention of single tokens to a short cache: one question of 20 tokens, latency only
        dict(name="attend-short", op="attend", batch=1, rows=1, heads=12, group=1, cap=64, held=20, ragged=False, tail=12, fmt="e4m3", dtype="bf16", seed=4),
        # a decode step of 64 questions with five beams each over the 100 x 100 prefix; each beam's own steps are in the tail
        dict(name="attend-beams", op="attend", batch=64, rows=5, heads=12, group=1, cap=10176, held=10120, ragged=True, tail=12, fmt="e4m3", dtype="bf16", seed=5),
        # the 12 answer rows of two questions at once, in fp32
        dict(name="attend-rows-fp32", op="attend", batch=2, rows=12, heads=12, group=1, cap=7168, held=7136, ragged=True, tail=12, fmt="int8", dtype="fp32", seed=6),
        # one token each of two long documents, four query heads to a key head
        dict(name="attend-long-grouped", op="attend", batch=2, rows=1, heads=8, group=4, cap=131072, held=131017, ragged=False, tail=0, fmt="int8", dtype="bf16", seed=7),
        # selection for one question: five beams over 5 000 words and 20 frames x 30 OCR slots
        dict(name="select-one", op="select", batch=1, beams=5, select=5, vocab=5600, dtype="fp32", finished=0.0, masked=0.0, seed=8),
        # a batch of 64 over 5 000 words and 100 x 100 OCR slots; some beams have ended, some slots are masked
        dict(name="select-batch", op="select", batch=64, beams=5, select=5, vocab=15000, dtype="fp32", finished=0.2, masked=0.3, seed=9),
        # a text vocabulary of 30 522 in bf16, eight beams, twice as many candidates as beams
        dict(name="select-text", op="select", batch=48, beams=8, select=16, vocab=30522, dtype="bf16", finished=0.1, masked=0.0, seed=10),
        # the states of five beams: keys and values of 12 steps in three layers
        dict(name="reorder-states", op="reorder", batch=64, beams=5, outer=3, steps=12, used=12, width=1536, dtype="bf16", seed=11),
        # the token lists of four beams, an odd number of steps, 8-byte elements
        dict(name="reorder-tokens", op="reorder", batch=48, beams=4, outer=1, steps=13, used=13, width=1, dtype="int64", seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "select", "select", "reorder"])
    c = dict(op=op, seed=rng.randrange(1 << 30))
    if op == "append":
        c["batch"] = _log_int(rng, 1, 64)
        c["heads"] = rng.choice([1, 3, 8, 12, 16])
        # tokens already held, and new ones; at most the largest listed case's total
        most = 10120 * 64 * 12 // (c["batch"] * c["heads"])
        c["new"] = min(_log_int(rng, 1, 10120), most // 2)
        c["held"] = min(_log_int(rng, 1, 5000) - 1, most // 2)
        c["cap"] = -(-(c["held"] + c["new"] + rng.randrange(0, 80)) // BLOCK) * BLOCK
        c["fmt"], c["dtype"] = rng.choice(["int8", "e4m3"]), rng.choice(["bf16", "bf16", "fp32"])
        c["fused"], c["listed_rows"] = rng.random() < 0.5, rng.random() < 0.5
    elif op == "attend":
        c["batch"] = _log_int(rng, 1, 64)
        c["rows"] = rng.choice([1, 1, 2, 3, 4, 5, 8, 12, 16])
        c["heads"], c["group"] = rng.choice([(12, 1), (16, 1), (12, 1), (8, 4), (2, 6), (1, 12), (3, 5)])
        most = min(131072, 10120 * 64 * 12 // (c["batch"] * c["heads"]))
        c["held"] = min(_log_int(rng, 1, 131072), most)
        c["cap"] = -(-(c["held"] + rng.randrange(0, 80)) // BLOCK) * BLOCK
        c["ragged"] = rng.random() < 0.6
        c["tail"] = rng.choice([0, 1, 7, 12, 33])
        c["fmt"], c["dtype"] = rng.choice(["int8", "e4m3"]), rng.choice(["bf16", "bf16", "fp32"])
    elif op == "select":
        c["batch"] = _log_int(rng, 1, 64)
        c["beams"] = rng.choice([1, 2, 3, 4, 5, 8, 13])
        c["vocab"] = min(_log_int(rng, 50, 130000), 12_000_000 // (c["batch"] * c["beams"]))
        c["select"] = rng.choice([c["beams"], c["beams"], 2 * c["beams"]])
        c["dtype"] = rng.choice(["fp32", "fp32", "bf16"])
        c["finished"], c["masked"] = rng.choice([0.0, 0.1, 0.3]), rng.choice([0.0, 0.0, 0.3, 0.9])
    else:
        c["batch"] = _log_int(rng, 1, 64)
        c["beams"] = rng.choice([1, 2, 3, 4, 5, 8, 13, 16])
        c["outer"] = rng.choice([1, 2, 3, 6])
        c["steps"] = rng.randrange(1, 41)
        c["used"] = rng.randrange(1, c["steps"] + 1)
        c["width"] = rng.choice([1, 3, 50, 64, 768, 1536])
        c["dtype"] = rng.choice(["bf16", "bf16", "fp32", "int64"])
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------

def _key_rows(shape, g, dev):
    """Rows like a trained projection's: a fixed offset and a spread for each channel, a normal rest."""
    ch = torch.randn(shape[-2:], generator=g, device=dev)
    x = torch.randn(shape, generator=g, device=dev)
    return x.mul_(0.3 + 0.4 * torch.rand(shape[-2:], generator=g, device=dev)).add_(0.5 * ch)


def _scale(amax, fmt):
    amax = amax.clamp(min=TINY)
    if fmt == "int8":
        return (amax.double() / 127.0).float()
    part, e = torch.frexp(amax)                                          # amax = part 2^e, part in [1/2, 1); 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(amax), e - 9 + (part > 0.875))


def _round_codes(x, s, fmt):
    if fmt == "e4m3":
        return (x * s.reciprocal()).to(torch.float8_e4m3fn)              # a power of two: the product is exact
    return torch.round(x.double() * s.double().reciprocal().float().double()).to(torch.int8)


def _spread(s, cap):
    """[B, H, nblk] -> [B, H, cap, 1]: each block's scale at each of its tokens."""
    return s.repeat_interleave(BLOCK, dim=2)[:, :, :cap].unsqueeze(-1)


def _codes(x, held, fmt):
    """Codes and scales of x [B, H, cap, 64] fp32, tokens behind ``held`` [B] empty (code 0)."""
    B, H, cap, _ = x.shape
    there = (torch.arange(cap, device=x.device) < held[:, None])[:, None, :, None]
    x = torch.where(there, x, torch.zeros((), device=x.device))
    s = _scale(x.abs().view(B, H, cap // BLOCK, BLOCK * HD).amax(-1), fmt)
    return _round_codes(x, _spread(s, cap), fmt), s


def _stored_v(v8):
    """Codes [B, H, cap, 64] -> the cache's storage order [B, H, nblk, 64 dims, 64 positions]."""
    B, H, cap, _ = v8.shape
    raw = v8.view(torch.uint8).view(B, H, cap // BLOCK, BLOCK, HD)
    return raw[:, :, :, ORDER].transpose(3, 4).contiguous().view(v8.dtype)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + case["seed"])
    op = case["op"]
    if op in ("append", "attend"):
        B, H, cap, held, fmt = case["batch"], case["heads"], case["cap"], case["held"], case["fmt"]
        dt = DTYPE[case["dtype"]]
        if op == "append" or case["ragged"]:
            low = 0 if op == "append" else 1
            lens = torch.randint(min(low, held), held + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            lens[0] = held
        else:
            lens = torch.full((B,), held, dtype=torch.int32, device=dev)
        st = dict(op=op, fmt=fmt, lens=lens, cap=cap)
        for name in ("k", "v"):
            x = _key_rows((B, cap, H, HD), g, dev).transpose(1, 2) if held else torch.zeros(B, H, cap, HD, device=dev)
            codes, s = _codes(x.contiguous(), lens, fmt)
            st[name + "8"], st[name + "s"] = codes, s
        st["k_stored"] = st["k8"].view(B, H, cap // BLOCK, BLOCK, HD).clone()
        st["v_stored"] = _stored_v(st["v8"])
        if own:
            # the handle that a program keeps over the steps of a decode; it takes the tensors as they are
            from vitxt_gqa_amd import decode
            st["cache"] = decode.KVCache8.from_parts(st.pop("k_stored"), st.pop("v_stored"), st["ks"].clone(), st["vs"].clone(), lens.clone())
    if op == "append":
        T = case["new"]
        if case["fused"]:
            # the fused Q | K | V projection of a layer; keys and values are slices of its rows
            qkv = torch.empty(B, T, 3, H, HD, dtype=dt, device=dev)
            qkv[:, :, 0] = 0.0
            qkv[:, :, 1] = _key_rows((B, T, H, HD), g, dev)
            qkv[:, :, 2] = _key_rows((B, T, H, HD), g, dev)
            st["k"], st["v"] = qkv[:, :, 1], qkv[:, :, 2]
        else:
            st["k"], st["v"] = _key_rows((B, T, H, HD), g, dev).to(dt), _key_rows((B, T, H, HD), g, dev).to(dt)
        st["counts"] = st["rows"] = None
        if case["listed_rows"]:
            # the visible rows of each sequence, ascending, and how many they are
            seen = torch.rand(B, T, generator=g, device=dev) < 0.7
            seen[:, 0] = True
            st["counts"] = seen.sum(1, dtype=torch.int32)
            st["rows"] = torch.argsort((~seen).to(torch.uint8), dim=1, stable=True).to(torch.int32)
        elif T > 1:
            st["counts"] = torch.randint(1, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    elif op == "attend":
        N, G, T = case["rows"], case["group"], case["tail"]
        st["q"] = (1.5 * torch.randn(B, N, H * G, HD, generator=g, device=dev)).to(dt)
        st["tail_k"] = st["tail_v"] = st["tail_len"] = None
        if T:
            st["tail_k"], st["tail_v"] = _key_rows((B, N, T, H, HD), g, dev).to(dt), _key_rows((B, N, T, H, HD), g, dev).to(dt)
            st["tail_len"] = torch.randint(0, T + 1, (B, N), generator=g, device=dev, dtype=torch.int32)
    elif op == "select":
        B, N, V = case["batch"], case["beams"], case["vocab"]
        x = 2.0 * torch.randn(B, N, V, generator=g, device=dev)
        if case["masked"] > 0:
            x = x.masked_fill(torch.rand(B, N, V, generator=g, device=dev) < case["masked"], -math.inf)
        st = dict(op=op, n=case["select"], pad=min(2, V - 1), logits=x.to(DTYPE[case["dtype"]]))
        st["scores"] = -torch.sort(6.0 * torch.rand(B, N, generator=g, device=dev), dim=1).values
        st["finished"] = torch.rand(B, N, generator=g, device=dev) < case["finished"] if case["finished"] > 0 else None
    elif op == "reorder":
        B, N = case["batch"], case["beams"]
        shape = (case["outer"], B, N, case["steps"], case["width"])
        if case["dtype"] == "int64":
            x = torch.randint(0, 15000, shape, generator=g, device=dev)
        else:
            x = torch.randn(shape, generator=g, device=dev).to(DTYPE[case["dtype"]])
        st = dict(op=op, x=x, used=case["used"], parents=torch.randint(0, N, (B, N), generator=g, device=dev))
    return st


# ---- the plain forms --------------------------------------------------------------------------------------------------------------------

def _append_plain(codes, s_old, lens, x, counts, rows, fmt, out_dtype):
    """-> (the values the block codes stand for after the append [B, H, cap, 64], scales)."""
    B, H, cap, _ = codes.shape
    dev = codes.device
    T = rows.shape[1] if rows is not None else x.shape[1]
    n = counts.long() if counts is not None else torch.full((B,), T, device=dev)
    t = torch.arange(cap, device=dev)[None, :]
    held = lens.long()[:, None]
    is_new = (t >= held) & (t < held + n[:, None])                                                  # [B, cap]
    src = (t - held).clamp(0, T - 1)
    if rows is not None:
        src = torch.gather(rows.long(), 1, src)
    new = x.gather(1, src[:, :, None, None].expand(B, cap, H, HD)).transpose(1, 2).float()          # [B, H, cap, 64]
    old = codes.float() * _spread(s_old, cap)
    both = torch.where(is_new[:, None, :, None], new, torch.where((t < held)[:, None, :, None], old, torch.zeros((), device=dev)))
    amax = torch.where(is_new[:, None, :, None], new, torch.zeros((), device=dev)).abs().reshape(B, H, cap // BLOCK, -1).amax(-1)
    touched = is_new.view(B, cap // BLOCK, BLOCK).any(-1)[:, None]
    keeps = (t < held).view(B, cap // BLOCK, BLOCK).any(-1)[:, None]
    s = _scale(amax, fmt)
    s = torch.where(touched, torch.where(keeps, torch.maximum(s, s_old), s), s_old)
    now = torch.where(touched.repeat_interleave(BLOCK, 2).unsqueeze(-1), _round_codes(both, _spread(s, cap), fmt).float(), codes.float())
    values = torch.where((t < held + n[:, None])[:, None, :, None], now * _spread(s, cap), torch.zeros((), device=dev))
    return values.to(out_dtype), s


def _attend_plain(st):
    q, lens = st["q"], st["lens"]
    B, N, HQ, _ = q.shape
    _, H, cap, _ = st["k8"].shape
    G = HQ // H
    k = st["k8"].float() * _spread(st["ks"], cap)
    v = st["v8"].float() * _spread(st["vs"], cap)
    qf = q.float().view(B, N, H, G, HD).permute(0, 2, 1, 3, 4).reshape(B, H, N * G, HD)
    s = torch.matmul(qf, k.transpose(2, 3)) * 0.125
    s = s.masked_fill((torch.arange(cap, device=q.device) >= lens[:, None])[:, None, None, :], -math.inf)
    if st["tail_k"] is not None:
        T = st["tail_k"].shape[2]
        tk = st["tail_k"].float().permute(0, 3, 1, 2, 4)                                             # [B, H, N, T, 64]
        tv = st["tail_v"].float().permute(0, 3, 1, 2, 4)
        ts = torch.matmul(qf.view(B, H, N, G, HD), tk.transpose(3, 4)) * 0.125                       # [B, H, N, G, T]
        ts = ts.masked_fill((torch.arange(T, device=q.device) >= st["tail_len"][:, :, None])[:, None, :, None, :], -math.inf)
        s = torch.cat([s, ts.reshape(B, H, N * G, T)], dim=3)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros((), device=q.device), m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :cap], v)
    if st["tail_k"] is not None:
        o = o + torch.matmul(p[..., cap:].view(B, H, N, G, T), tv).view(B, H, N * G, HD)
    o = torch.where(l > 0, o / l, torch.zeros((), device=q.device))
    lse = (m + torch.log(l)).squeeze(-1)
    back = lambda x, d: x.view(B, H, N, G, *d).transpose(1, 2).reshape(B, N, HQ, *d)
    return back(o, (HD,)).to(q.dtype), back(lse, ())


def _select_plain(st):
    x = st["logits"].double()
    B, N, V = x.shape
    m = x.amax(-1, keepdim=True).clamp(min=-1e300)                                                   # (a row without a word left)
    d = x - m
    logp = torch.where(x > -math.inf, d - torch.log(torch.exp(d).sum(-1, keepdim=True)), x)
    if st["finished"] is not None:
        ended = torch.full((V,), -math.inf, dtype=torch.float64, device=x.device)
        ended[st["pad"]] = 0.0
        logp = torch.where(st["finished"][..., None], ended, logp)
    total = (st["scores"].double()[..., None] + logp).view(B, N * V)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :st["n"]], at[:, :st["n"]]
    return best.float(), at // V, at % V


def run(st):
    op = st["op"]
    if own:
        from vitxt_gqa_amd import decode
        if op == "append":
            cache = st["cache"]
            cache.set_lens(st["lens"])
            cache.append(st["k"], st["v"], counts=st["counts"], rows=st["rows"])
            return (*cache.dequantize(st["k"].dtype), cache.k_scale, cache.v_scale, cache.lens)
        if op == "attend":
            return decode.attend(st["q"], st["cache"], st["tail_k"], st["tail_v"], st["tail_len"], scale=0.125)
        if op == "select":
            return decode.beam_select(st["logits"], st["scores"], st["n"], finished=st["finished"], pad=st["pad"])
        return decode.beam_reorder(st["x"], st["parents"], batch_dim=1, used=st["used"])
    if op == "append":
        dt = st["k"].dtype
        k, ks = _append_plain(st["k8"], st["ks"], st["lens"], st["k"], st["counts"], st["rows"], st["fmt"], dt)
        v, vs = _append_plain(st["v8"], st["vs"], st["lens"], st["v"], st["counts"], st["rows"], st["fmt"], dt)
        new = st["counts"] if st["counts"] is not None else st["k"].shape[1]
        return k, v, ks, vs, st["lens"] + new
    if op == "attend":
        return _attend_plain(st)
    if op == "select":
        return _select_plain(st)
    x, u = st["x"], st["used"]
    at = st["parents"][None, :, :, None, None].expand(x.shape[0], -1, -1, u, x.shape[4])
    x[:, :, :, :u] = torch.gather(x[:, :, :, :u], 2, at)
    return x


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp32": 4, "int64": 8}[case["dtype"]]
    if op == "append":
        B, H = case["batch"], case["heads"]
        new = case["new"] if case["new"] == 1 else case["new"] * (0.7 if case["listed_rows"] else 0.5)
        held = case["held"] * 0.5
        blocks = case["cap"] // BLOCK
        # new rows read once, their codes written; the read-back reads every code held and writes every value of the capacity
        each = new * HD * (size + 1) + (held + new) * HD + case["cap"] * HD * size + 3 * blocks * 4
        return {"bytes": 2 * B * H * each, "flops": 2 * B * H * HD * (3 * new + held)}
    if op == "attend":
        B, H, N, G = case["batch"], case["heads"], case["rows"], case["group"]
        held = case["held"] * (0.5 if case["ragged"] else 1.0)
        tail = case["tail"] * 0.5
        b = B * H * (2 * held * HD + 2 * held / BLOCK * 4 + 2 * N * tail * HD * size) + B * N * H * G * (2 * HD * size + 4)
        return {"bytes": b, "flops": 4 * B * N * H * G * HD * (held + tail)}
    if op == "select":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * (1 - case["finished"]) * size + case["batch"] * (case["beams"] * 5 + case["select"] * 20), "flops": 3 * n}
    # a beam that keeps its place has nothing to move: 1 in N of a random draw
    n = case["outer"] * case["batch"] * case["beams"] * case["used"] * case["width"]
    return {"bytes": max(2 * n * size * (1 - 1 / case["beams"]), 8 * case["batch"] * case["beams"]), "flops": 0}


# ---- 64 bits ------------------------------------------------------------------------------------------------------------------------------

def _e4m3(x):
    """|x| <= 448 in 64 bits to the nearest e4m3 number, ties to even: 3 fraction bits, least exponent -6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    def append64(codes, s_old, lens, x, counts, rows, fmt):
        out, scales = [], []
        B, H, cap, _ = codes.shape
        for b in range(B):
            held = int(lens[b])
            n = int(counts[b]) if counts is not None else x.shape[1]
            src = rows[b, :n].long() if rows is not None else torch.arange(n, device=x.device)
            val = torch.zeros(H, cap, HD, dtype=torch.float64, device=x.device)
            s = s_old[b].double().clone()
            val[:, :held] = codes[b, :, :held].double() * s.repeat_interleave(BLOCK, 1)[:, :held, None]
            val[:, held:held + n] = x[b, src].transpose(0, 1).double()
            first, last = held // BLOCK, (held + n - 1) // BLOCK
            fresh = val.clone()
            fresh[:, :held] = 0.0
            got = fresh[:, first * BLOCK:(last + 1) * BLOCK].abs().reshape(H, last - first + 1, -1).amax(-1).clamp(min=TINY)
            if fmt == "int8":
                got = (got / 127.0).float().double()                        # the scale is held in 32 bits
            else:
                got = torch.exp2(torch.ceil(torch.log2(got / 448.0) - 1e-13))
            if held % BLOCK:
                got[:, 0] = torch.maximum(got[:, 0], s[:, first])
            s[:, first:last + 1] = got
            each = got.repeat_interleave(BLOCK, 1)[..., None]
            part = val[:, first * BLOCK:(last + 1) * BLOCK] * (1.0 / each).float().double()
            val[:, first * BLOCK:(last + 1) * BLOCK] = (torch.round(part) if fmt == "int8" else _e4m3(part)) * each
            out.append(val)
            scales.append(s)
        return torch.stack(out), torch.stack(scales)

    op = case["op"]
    st = prepare(case, seed)
    if op == "append":
        if case["batch"] * case["heads"] * case["cap"] > 40_000_000:
            return None
        k, ks = append64(st["k8"], st["ks"], st["lens"], st["k"], st["counts"], st["rows"], st["fmt"])
        v, vs = append64(st["v8"], st["vs"], st["lens"], st["v"], st["counts"], st["rows"], st["fmt"])
        return k, v, ks, vs, None
    if op == "attend":
        q = st["q"].double() * 0.125
        B, N, HQ, _ = q.shape
        H = st["k8"].shape[1]
        G = HQ // H
        out = torch.zeros(B, N, HQ, HD, dtype=torch.float64, device=q.device)
        lse = torch.empty(B, N, HQ, dtype=torch.float64, device=q.device)
        for b in range(B):
            n = int(st["lens"][b])
            ks = st["ks"][b].double().repeat_interleave(BLOCK, 1)[:, :n, None]
            vs = st["vs"][b].double().repeat_interleave(BLOCK, 1)[:, :n, None]
            k, v = st["k8"][b, :, :n].double() * ks, st["v8"][b, :, :n].double() * vs                # [H, n, 64]
            qb = q[b].view(N, H, G, HD).transpose(0, 1).reshape(H, N * G, HD)
            sc = torch.bmm(qb, k.transpose(1, 2).contiguous()).view(H, N, G, n)
            if st["tail_k"] is not None:
                T = st["tail_k"].shape[2]
                tk, tv = st["tail_k"][b].double().permute(2, 0, 1, 3), st["tail_v"][b].double().permute(2, 0, 1, 3)      # [H, N, T, 64]
                ts = (qb.view(H, N, G, 1, HD) * tk[:, :, None]).sum(-1)
                ts = ts.masked_fill(torch.arange(T, device=q.device) >= st["tail_len"][b][None, :, None, None], -math.inf)
                sc = torch.cat([sc, ts], dim=3)
            e = torch.logsumexp(sc, dim=3)
            p = torch.where(e[..., None] > -math.inf, torch.exp(sc - e[..., None]), torch.zeros((), dtype=torch.float64, device=q.device))
            o = torch.bmm(p[..., :n].reshape(H, N * G, n).contiguous(), v).view(H, N, G, HD)
            if st["tail_k"] is not None:
                o = o + (p[..., n:, None] * tv[:, :, None]).sum(3)
            out[b] = o.transpose(0, 1).reshape(N, HQ, HD)
            lse[b] = e.transpose(0, 1).reshape(N, HQ)
        return out, lse
    if op == "select":
        x, cum = st["logits"].double(), st["scores"].double()
        B, N, V = x.shape
        norm = torch.logsumexp(x, dim=2)
        best = torch.empty(B, st["n"], dtype=torch.float64, device=x.device)
        for b in range(B):
            rows = cum[b][:, None] + torch.where(x[b] > -math.inf, x[b] - norm[b][:, None], x[b])
            if st["finished"] is not None:
                for i in torch.nonzero(st["finished"][b]).flatten().tolist():
                    rows[i] = -math.inf
                    rows[i, st["pad"]] = cum[b, i]
            best[b] = torch.topk(rows.flatten(), st["n"]).values
        return best, None, None
    if st["x"].dtype == torch.int64:
        return None
    x, u = st["x"], st["used"]
    want = x.double()
    for b in range(x.shape[1]):
        for i, p in enumerate(st["parents"][b].tolist()):
            want[:, b, i, :u] = x[:, b, p, :u].double()
    return want
