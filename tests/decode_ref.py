"""Plain 64-bit statements of the decode operators (vitxt_gqa_amd/decode.py), on the CPU."""
import math

import torch

BLOCK, HD = 64, 64
ORDER = [((p >> 2) & 3) * 16 + (p >> 4) * 4 + (p & 3) for p in range(BLOCK)]      # position p of a value row holds this token
QMAX = {"int8": 127.0, "e4m3": 448.0}


def round_e4m3(x):
    """To the nearest e4m3 number, ties to even (|x| <= 448): 3 fraction bits, least exponent -6."""
    x = x.double()
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def scale_of(amax, fmt):
    """fp32 scale of a block whose largest magnitude is ``amax`` (fp32)."""
    amax = amax.float().clamp(min=2.0 ** -100)
    if fmt == "int8":
        return (amax.double() / 127.0).float()
    s = torch.exp2(torch.ceil(torch.log2(amax.double() / 448.0) - 1e-12))
    return s.float()


def codes_of(x, s, fmt):
    """Code values (double) of x under the fp32 scales s."""
    y = x.double() * (1.0 / s.double()).float().double()
    return torch.round(y).clamp(-127, 127) if fmt == "int8" else round_e4m3(y.clamp(-448, 448))


class RefCache:
    """The cache as lists of fp32 values: code values [B][H] of tokens, scales per block."""

    def __init__(self, B, H, fmt):
        self.B, self.H, self.fmt = B, H, fmt
        self.codes = [[[torch.zeros(0, HD, dtype=torch.float64) for _ in range(H)] for _ in range(B)] for _ in range(2)]
        self.scales = [[[[] for _ in range(H)] for _ in range(B)] for _ in range(2)]

    def lens(self):
        return [self.codes[0][b][0].shape[0] for b in range(self.B)]

    def truncate(self, lens):
        for kv in range(2):
            for b in range(self.B):
                for h in range(self.H):
                    self.codes[kv][b][h] = self.codes[kv][b][h][:lens[b]]
                    self.scales[kv][b][h] = self.scales[kv][b][h][:-(-lens[b] // BLOCK)]

    def append(self, k, v, counts=None, rows=None):
        for kv, x in enumerate((k.cpu().float(), v.cpu().float())):
            for b in range(self.B):
                T = rows.shape[1] if rows is not None else x.shape[1]
                n = max(0, min(T, int(counts[b]))) if counts is not None else T
                src = [int(rows[b, j]) if rows is not None else j for j in range(n)]
                for h in range(self.H):
                    new = x[b, src, h] if n else torch.zeros(0, HD)
                    codes, scales = self.codes[kv][b][h], self.scales[kv][b][h]
                    at = 0
                    while at < n:
                        held = codes.shape[0]
                        take = min(n - at, BLOCK - held % BLOCK)
                        part = new[at:at + take]
                        if torch.isfinite(part).all():
                            s = scale_of(part.abs().max(), self.fmt)
                        else:
                            s = torch.tensor(math.nan)
                        if held % BLOCK:
                            first = held - held % BLOCK
                            s_old = torch.tensor(scales[-1])
                            s = torch.maximum(s, s_old)                              # NaN on either side stays
                            old = codes[first:] * s_old.double()
                            old = old.float()                                        # code * scale as an fp32 number
                            again = codes_of(old, s, self.fmt) if s == s else torch.zeros_like(codes[first:])
                            codes = torch.cat([codes[:first], again])
                            scales[-1] = float(s)
                        else:
                            scales.append(float(s))
                        codes = torch.cat([codes, codes_of(part, s, self.fmt) if s == s else torch.zeros(take, HD, dtype=torch.float64)])
                        at += take
                    self.codes[kv][b][h] = codes

    def values(self, kv, b, h):
        """fp64 values of the tokens held."""
        c, s = self.codes[kv][b][h], torch.tensor(self.scales[kv][b][h], dtype=torch.float64)
        return c * s.repeat_interleave(BLOCK)[:c.shape[0], None]


def read_cache(cache):
    """(keys, values) fp64 lists [b][h] of a KVCache8's storage, by the documented layout."""
    lens = cache.lens.tolist()
    k = cache.k.cpu().to(torch.float32).double() * cache.k_scale.cpu().double()[..., None, None]
    v = cache.v.cpu().to(torch.float32).double() * cache.v_scale.cpu().double()[..., None, None]
    B, H, n = k.shape[:3]
    k = k.reshape(B, H, n * BLOCK, HD)
    vt = torch.empty_like(v)
    vt[:, :, :, ORDER] = v.transpose(3, 4)                                           # [.., dim, position] -> [.., token, dim]
    v = vt.reshape(B, H, n * BLOCK, HD)
    return [[(k[b, h, :lens[b]], v[b, h, :lens[b]]) for h in range(H)] for b in range(B)]


def attend_ref(q, kv, tail_k=None, tail_v=None, tail_len=None, scale=0.125):
    """kv[b][h] = (keys, values) fp64.  -> out, lse (fp64), smax: largest sum of |q_d k_d| * scale, vmax: largest |v|."""
    q = q.cpu().double()
    B, N, HQ, _ = q.shape
    H = len(kv[0])
    G = HQ // H
    out, lse = torch.zeros(B, N, HQ, HD, dtype=torch.float64), torch.full((B, N, HQ), -math.inf, dtype=torch.float64)
    smax = vmax = 0.0
    for b in range(B):
        for n in range(N):
            for i in range(HQ):
                k, v = kv[b][i // G]
                if tail_k is not None:
                    t = tail_k.shape[2] if tail_len is None else max(0, min(tail_k.shape[2], int(tail_len[b, n])))
                    k = torch.cat([k, tail_k[b, n, :t, i // G].cpu().double()])
                    v = torch.cat([v, tail_v[b, n, :t, i // G].cpu().double()])
                if not len(k):
                    continue
                s = (k @ q[b, n, i]) * scale
                lse[b, n, i] = torch.logsumexp(s, 0)
                out[b, n, i] = torch.softmax(s, 0) @ v
                smax = max(smax, float((k.abs() @ q[b, n, i].abs()).max()) * abs(scale))
                vmax = max(vmax, float(v.abs().max()))
    return out, lse, smax, vmax


def select_ref(logits, scores, K, finished=None, pad=0):
    """-> scores fp64 [B, K], parents, tokens."""
    x = logits.cpu().double()
    x = torch.where(torch.isnan(x), torch.tensor(-math.inf, dtype=torch.float64), x).clamp(max=torch.finfo(torch.float32).max)
    B, N, V = x.shape
    cum = scores.cpu().double()
    cum = torch.where(torch.isnan(cum), torch.tensor(-math.inf, dtype=torch.float64), cum)
    # relative to the row's maximum: beside a mask of -3.4e38 the logarithm of a sum would vanish even in 64 bits
    top = x.amax(2, keepdim=True).clamp(min=-1e300)
    lp = torch.where(x > -math.inf, (x - top) - torch.logsumexp(x - top, 2, keepdim=True), torch.full_like(x, -math.inf))
    if finished is not None:
        only = torch.full((V,), -math.inf, dtype=torch.float64)
        only[pad] = 0.0
        lp = torch.where(finished.cpu().bool()[..., None], only, lp)
    total = (cum[..., None] + lp).reshape(B, N * V)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    return best[:, :K + 1], at[:, :K] // V, at[:, :K] % V
