"""The decode operators (vitxt_gqa_amd/decode.py) against plain 64-bit statements (decode_ref.py).

Tolerances, u = 2^-24 (half an fp32 step), w = 2^-8 (half a bf16 step):
  append        none: codes and scales are defined by exact products
  attend        a score is 64 products (each exact: <= 8 x 8 significant bits; three terms of an fp32 query) summed in fp32 by the matrix pipe, then two
                rescalings: |d score| <= 200 u S, S = scale * max sum |q_d k_d|.  out: 2 |d score| vmax from the weights, the sums over tokens and shares
                (L / 32 + 64) u vmax, probabilities held in f16 (bf16 results: off by 2^-12 of themselves, or where they are subnormal by 2^-25 of
                the largest, so by (2^-12 + L 2^-25) vmax over a row) or in 24 bits (fp32: u vmax), one rounding of the result (bf16: w |out|).
                lse: |d score| + (L / 32 + 64) u + u |lse|
  beam_select   the order is the 64-bit statement's wherever neighbours differ by more than the tolerance (and where they are equal); a score's
                error is that of log sum exp: terms e^d with d rounded in fp32 (104 u at most before they vanish) and summed: 160 u, + u |score|
"""
import math

import pytest
import torch

from decode_ref import BLOCK, HD, RefCache, attend_ref, read_cache, select_ref

gpu = pytest.mark.gpu
pytestmark = gpu
U, W = 2.0 ** -24, 2.0 ** -8
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _rows(g, *shape, dtype=torch.float32):
    """Rows with a fixed offset per channel, spreads that differ by channel, and some values far out."""
    x = torch.randn(*shape, generator=g) * (0.2 + torch.rand(shape[-1], generator=g)) + torch.randn(shape[-1], generator=g) * 0.5
    x = torch.where(torch.rand(*shape, generator=g) < 0.002, x * 8, x)
    return x.to(dtype)


def _same_cache(cache, ref):
    assert cache.lens.tolist() == ref.lens()
    got = read_cache(cache)
    for b in range(ref.B):
        for h in range(ref.H):
            for kv in range(2):
                want = ref.values(kv, b, h)
                assert torch.equal(got[b][h][kv].nan_to_num(nan=1e30), want.nan_to_num(nan=1e30)), (b, h, kv)


def _check_attend(q, cache, tail_k=None, tail_v=None, tail_len=None, scale=0.125, got=None):
    from vitxt_gqa_amd import decode
    dev = q.device
    out, lse = got if got is not None else decode.attend(q, cache, tail_k, tail_v, None if tail_len is None else tail_len.to(dev), scale)
    ref, rlse, S, vmax = attend_ref(q, read_cache(cache), tail_k, tail_v, tail_len, scale)
    L = cache.capacity
    ds = 200 * U * S
    terms = (2.0 ** -12 + L * 2.0 ** -25 if q.dtype == torch.bfloat16 else U) + (L / 32 + 64) * U
    tol = (2 * ds + terms) * vmax + (W if q.dtype == torch.bfloat16 else U) * ref.abs() + 1e-30
    err = (out.cpu().double() - ref).abs()
    assert out.dtype == q.dtype and bool((err <= tol).all()), "out off by %.3g of %.3g" % (err.max(), tol.max())
    empty = rlse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty) and bool((out.cpu()[empty] == 0).all())
    e2 = (lse.cpu().double() - rlse)[~empty].abs()
    t2 = (ds + (L / 32 + 64) * U + U * rlse.abs())[~empty]
    assert bool((e2 <= t2).all()), "lse off by %.3g" % e2.max()
    return out, lse


# ---- append ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [[1], [63], [64], [65], [130], [1, 1, 62, 1, 3], [64, 5, 128], [40] * 4])
def test_append_is_exact(fmt, dtype, new):
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(len(new) * 1000 + new[0])
    B, H = 3, 2
    cache, ref = decode.KVCache8(B, H, sum(new), fmt), RefCache(B, H, fmt)
    for i, T in enumerate(new):
        k, v = _rows(g, B, T, H, HD, dtype=DT[dtype]) * (1.0 + 0.7 * i), _rows(g, B, T, H, HD, dtype=DT[dtype])        # (scales grow from part to part)
        cache.append(k.cuda(), v.cuda())
        ref.append(k, v)
        _same_cache(cache, ref)
    for dt, half in ((torch.float32, U), (torch.bfloat16, W)):
        kk, vv = cache.dequantize(dt)
        for kv, x in enumerate((kk, vv)):
            assert x.dtype == dt and x.shape == (B, H, cache.capacity, HD)
            for b in range(B):
                for h in range(H):
                    want = ref.values(kv, b, h)
                    assert bool(((x[b, h, :len(want)].cpu().double() - want).abs() <= half * want.abs()).all())
                    assert not x[b, h, len(want):].any()


@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "fp32")])
def test_append_listed_rows_ragged_counts(fmt, dtype):
    """Rows of a fused projection by a list, counts from 0 to more than T, three times over (blocks joined at odd places)."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(5)
    B, H, R, T = 5, 3, 150, 97
    cache, ref = decode.KVCache8(B, H, 400, fmt), RefCache(B, H, fmt)
    for i in range(3):
        qkv = _rows(g, B, R, 3, H, HD, dtype=DT[dtype])
        rows = torch.stack([torch.randperm(R, generator=g)[:T] for _ in range(B)]).to(torch.int32)
        rows[1, :] = rows[1, 0]                                                              # the same row many times
        counts = torch.tensor([0, 1, 96, 97, 500][i:] + [-3, 40][:i], dtype=torch.int32)
        dev = qkv.cuda()
        wide = torch.zeros(B, T + 9, dtype=torch.int32).cuda()                                # rows with a longer batch stride
        wide[:, :T] = rows.cuda()
        cache.append(dev[:, :, 1], dev[:, :, 2], counts=counts.cuda(), rows=wide[:, :T])
        ref.append(qkv[:, :, 1], qkv[:, :, 2], counts, rows)
        _same_cache(cache, ref)


def test_append_orders_and_strides():
    """[B, H, T, 64] keys beside [B, T, H, 64] values, an expanded batch, a slice of wider rows."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(6)
    B, H, T = 2, 3, 70
    for k, v in ((_rows(g, B, H, T, HD).transpose(1, 2), _rows(g, B, T, H, HD)), (_rows(g, 1, T, H, HD).expand(B, -1, -1, -1), _rows(g, B, T, H, HD + 8)[..., 4:68])):
        cache, ref = decode.KVCache8(B, H, T), RefCache(B, H, "int8")
        kd = k.transpose(1, 2).contiguous().cuda().transpose(1, 2) if k.stride(1) == HD else k[:1].cuda().expand(B, -1, -1, -1)
        vd = v.cuda() if v.is_contiguous() else torch.nn.functional.pad(v, (4, 4)).cuda()[..., 4:68]
        cache.append(kd, vd)
        ref.append(k, v)
        _same_cache(cache, ref)
    assert cache.append(torch.zeros(B, 0, H, HD).cuda(), torch.zeros(B, 0, H, HD).cuda()) is cache and cache.lens.tolist() == [T, T]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_extremes(fmt):
    """Zeros, numbers below the smallest scale, one huge value, ties between codes."""
    from vitxt_gqa_amd import decode
    k = torch.zeros(1, 320, 1, HD)
    k[0, 64:128] = 1e-38
    k[0, 128:192] = 1.0
    k[0, 140, 0, 5] = 3e38
    k[0, 192:256, 0] = torch.arange(64)[:, None] * 0.5 + torch.arange(64) * 1.0           # many exact ties
    k[0, 256:320, 0] = torch.arange(64)[None] - 31.5
    k[0, 256, 0, 0] = 127.0 if fmt == "int8" else 448.0
    v = -k
    cache, ref = decode.KVCache8(1, 1, 320, fmt), RefCache(1, 1, fmt)
    cache.append(k.cuda(), v.cuda())
    ref.append(k, v)
    _same_cache(cache, ref)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_not_finite(bad):
    """A value that is not finite shows in its block of its head, keys or values, and nowhere else; also when a later append joins the block."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(7)
    B, H = 2, 2
    k, v = _rows(g, B, 100, H, HD), _rows(g, B, 100, H, HD)
    k[0, 70, 1, 3] = bad
    cache, ref = decode.KVCache8(B, H, 192), RefCache(B, H, "int8")
    for a, e in ((0, 90), (90, 100)):
        cache.append(k[:, a:e].cuda(), v[:, a:e].cuda())
        ref.append(k[:, a:e], v[:, a:e])
    _same_cache(cache, ref)
    s = cache.k_scale.cpu()
    assert torch.isnan(s[0, 1, 1]) and int(torch.isnan(s).sum()) == 1 and not torch.isnan(cache.v_scale).any()
    out, lse = decode.attend(_rows(g, B, 1, H, HD).cuda(), cache)
    assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(lse[0, 0, 1]) and int(torch.isnan(lse).sum()) == 1 and int(torch.isnan(out).sum()) == HD
    # a row the list does not name may hold anything
    cache.set_lens(0)
    k[0, 70, 1, 3], k[1, 20] = 0.0, bad
    rows = torch.tensor([[i for i in range(60) if i != 20]] * B, dtype=torch.int32)
    cache.append(k.cuda(), v.cuda(), rows=rows.cuda())
    assert not torch.isnan(cache.dequantize()[0][:, :, :59]).any()
    # a row number that is not there
    cache.set_lens(0)
    rows[1, 3] = 100
    rows[0, 5] = -1
    cache.append(v.cuda(), v.cuda(), rows=rows.cuda())
    assert torch.isnan(cache.k_scale[:, :, 0]).all() and torch.isnan(cache.v_scale[:, :, 0]).all()


def test_append_that_does_not_fit():
    """The sequence's length turns to -1, its results to NaN; the others are right; set_lens takes it back."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(8)
    B, H = 3, 2
    k, v = _rows(g, B, 70, H, HD), _rows(g, B, 70, H, HD)
    cache, ref = decode.KVCache8(B, H, 128), RefCache(B, H, "int8")
    n1, n2 = torch.tensor([70, 50, 70], dtype=torch.int32), torch.tensor([58, 70, 59], dtype=torch.int32)
    for n in (n1, n2):
        cache.append(k.cuda(), v.cuda(), counts=n.cuda())
    assert cache.lens.tolist() == [128, 120, -1]
    q = _rows(g, B, 1, H, HD).cuda()
    out, lse = decode.attend(q, cache)
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all() and not torch.isnan(out[:2]).any()
    assert torch.isnan(cache.dequantize()[0][2].float()).all()
    cache.append(k.cuda(), v.cuda(), counts=torch.zeros(B, dtype=torch.int32).cuda())
    assert cache.lens.tolist() == [128, 120, -1]
    cache.set_lens(torch.tensor([70, 50, 70], dtype=torch.int32).cuda())
    ref.append(k, v, n1)
    # (block 1 of the third sequence has been filled up since: its first 6 tokens were rounded again under the larger scale)
    assert cache.lens.tolist() == ref.lens()
    _check_attend(q, cache)


def test_append_leaves_the_rest_alone():
    from vitxt_gqa_amd import decode
    B, H, n = 2, 2, 4
    raw = [torch.full((B, H, n, BLOCK, HD), 77, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.full((B, H, n), 5.0, device="cuda") for _ in range(2)]
    cache = decode.KVCache8.from_parts(*raw, *scales, torch.tensor([64, 70], dtype=torch.int32, device="cuda"))
    x = torch.randn(B, 3, H, HD, device="cuda")
    cache.append(x, x, counts=torch.tensor([3, 0], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [67, 70]
    for r, s in zip(raw, scales):
        assert bool((r[1] == 77).all()) and bool((r[0, :, [0, 2, 3]] == 77).all()) and bool((s[1] == 5).all()) and bool((s[0, :, [0, 2, 3]] == 5).all())
        assert bool((s[0, :, 1] < 1).all())


# ---- attention -----------------------------------------------------------------------------------------------------------------------------
def _filled(g, B, H, lens, fmt="int8", cap=None, dtype=torch.float32):
    from vitxt_gqa_amd import decode
    T = max(max(lens), 1)
    cache = decode.KVCache8(B, H, cap or T, fmt)
    cache.append(_rows(g, B, T, H, HD, dtype=dtype).cuda(), _rows(g, B, T, H, HD, dtype=dtype).cuda(), counts=torch.tensor(lens, dtype=torch.int32).cuda())
    return cache


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,N,H,G,T", [
    ([1], 1, 1, 1, 0), ([0, 1, 63], 1, 2, 1, 0), ([64, 65, 0], 2, 1, 3, 5), ([20] * 2, 1, 12, 1, 12), ([700, 3, 511, 512], 5, 2, 1, 12), ([1000, 1], 3, 2, 6, 1),
    ([129, 640], 12, 1, 1, 12), ([300, 77], 16, 1, 1, 70), ([257], 17, 1, 1, 3), ([200, 0], 5, 1, 8, 130), ([0, 0], 2, 2, 1, 0), ([0, 5], 2, 2, 1, 4), ([2500], 33, 1, 2, 0)])
def test_attend(fmt, dtype, lens, N, H, G, T):
    g = torch.Generator().manual_seed(sum(lens) + N * 7 + G)
    B = len(lens)
    cache = _filled(g, B, H, lens, fmt)
    q = (_rows(g, B, N, H * G, HD) * 2).to(DT[dtype]).cuda()
    tk = tv = tl = None
    if T:
        tk, tv = (_rows(g, B, N, T, H, HD, dtype=DT[dtype]).cuda() for _ in range(2))
        tl = torch.randint(-1, T + 2, (B, N), generator=g, dtype=torch.int32)
        tl[0, 0] = 0
    _check_attend(q, cache, tk, tv, tl)


def test_attend_whole_tail_and_int_tail():
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(21)
    cache = _filled(g, 2, 2, [40, 0])
    q, tk, tv = _rows(g, 2, 3, 2, HD).cuda(), _rows(g, 2, 3, 9, 2, HD).cuda(), _rows(g, 2, 3, 9, 2, HD).cuda()
    _check_attend(q, cache, tk, tv)
    for t in (0, 4, 9, 50, -2):
        got = decode.attend(q, cache, tk, tv, t)
        _check_attend(q, cache, tk, tv, torch.full((2, 3), t, dtype=torch.int32), got=got)
    empty = torch.empty(2, 3, 0, 2, HD, device="cuda")
    assert torch.equal(decode.attend(q, cache, empty, empty)[0], decode.attend(q, cache)[0])
    out, lse = decode.attend(q[:, :0], cache)
    assert out.shape == (2, 0, 2, HD) and lse.shape == (2, 0, 2)


def test_attend_views():
    """Queries as a slice of fused rows, heads before rows, tails as slices of one [.., 2, H, 64] buffer and shared by the rows of a sequence (stride 0),
    lengths expanded."""
    g = torch.Generator().manual_seed(22)
    B, N, H, T = 2, 4, 3, 6
    cache = _filled(g, B, H, [130, 9], "e4m3")
    for dt in (torch.bfloat16, torch.float32):
        fused = _rows(g, B, N, 3, H, HD, dtype=dt).cuda()
        tail = _rows(g, B, 1, T, 2, H, HD, dtype=dt).cuda().expand(-1, N, -1, -1, -1, -1)
        tl = torch.arange(1, N + 1, dtype=torch.int32).expand(B, N)
        _check_attend(fused[:, :, 0], cache, tail[:, :, :, 0], tail[:, :, :, 1], tl)
        _check_attend(_rows(g, B, H, N, HD, dtype=dt).cuda().transpose(1, 2), cache)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,N,H,G,T", [
    ([300, 65], 40, 1, 1, 3), ([640, 1], 1, 1, 48, 20), ([200], 8, 2, 8, 0), ([129], 64, 1, 1, 33), ([500, 0], 65, 1, 1, 2), ([70], 9, 1, 16, 16), ([1500], 6, 1, 5, 0), ([40], 2, 1, 4, 17),
    ([40], 3, 1, 3, 17), ([1400], 43, 1, 3, 1), ([3000, 700], 5, 2, 1, 12), ([2600], 1, 2, 4, 0), ([1537, 1536, 1], 3, 1, 1, 5), ([1025, 1024], 2, 1, 2, 1), ([5000], 8, 3, 1, 40)])
def test_attend_row_groups(dtype, lens, N, H, G, T):
    """One to four 16-row tiles to a group and several groups, with a short cache (a single share) and a longer one, tails on either side of
    what a single share takes in."""
    g = torch.Generator().manual_seed(sum(lens) + N * 7 + G)
    cache = _filled(g, len(lens), H, lens, "int8" if N % 2 else "e4m3")
    q = (_rows(g, len(lens), N, H * G, HD) * 2).to(DT[dtype]).cuda()
    tk = tv = tl = None
    if T:
        tk, tv = (_rows(g, len(lens), N, T, H, HD, dtype=DT[dtype]).cuda() for _ in range(2))
        tl = torch.randint(0, T + 1, (len(lens), N), generator=g, dtype=torch.int32)
    _check_attend(q, cache, tk, tv, tl)


def test_attend_rows_do_not_touch_each_other():
    """A row of NaN or infinite queries, or with a NaN in its tail, leaves the other rows of its tile as they were."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(25)
    cache = _filled(g, 1, 2, [333])
    for dt in (torch.float32, torch.bfloat16):
        q = _rows(g, 1, 7, 4, HD, dtype=dt).cuda()
        tk, tv = (_rows(g, 1, 7, 6, 2, HD, dtype=dt).cuda() for _ in range(2))
        a, la = decode.attend(q, cache, tk, tv)
        q2, tk2, tv2 = q.clone(), tk.clone(), tv.clone()
        q2[0, 1] = math.nan
        q2[0, 3, 2, 5] = math.inf
        tv2[0, 4, 2, 1, 9] = math.nan
        tk2[0, 5, 5] = math.nan
        b, lb = decode.attend(q2, cache, tk2, tv2, 5)
        c, lc = decode.attend(q, cache, tk, tv, 5)
        bad = torch.zeros(1, 7, 4, HD, dtype=torch.bool)
        bad[0, 1] = bad[0, 3, 2] = True
        bad[0, 4, 2:, 9] = True
        bad = bad.cuda()
        assert bool(torch.isnan(b[bad]).all()) and torch.equal(b[~bad], c[~bad])
        _check_attend(q, cache, tk, tv, got=(a, la))
        _check_attend(q, cache, tk, tv, torch.full((1, 7), 5, dtype=torch.int32), got=(c, lc))


def test_attend_overflowing_scores_show():
    """Scores past fp32's range have no softmax in fp32: NaN, not a number made of the others."""
    from vitxt_gqa_amd import decode
    cache = decode.KVCache8(1, 1, 200)
    cache.append(torch.full((1, 200, 1, HD), 1e30).cuda(), torch.ones(1, 200, 1, HD).cuda())
    for dt in (torch.float32, torch.bfloat16):
        for N in (1, 12):
            out, lse = decode.attend(torch.full((1, N, 1, HD), 1e20, dtype=dt).cuda(), cache)
            assert bool(torch.isnan(out).all()) and not bool(torch.isfinite(lse).any())


def test_attend_tails_of_one_token_differ_in_strides_that_do_not_count():
    g = torch.Generator().manual_seed(24)
    cache = _filled(g, 1, 2, [100])
    k, v = _rows(g, 1, 3, 5, 2, HD).cuda(), _rows(g, 1, 3, 1, 2, HD).cuda()
    wide = torch.zeros(1, 3, 2, HD + 4, device="cuda")[..., :HD].unsqueeze(2)                   # odd steps of the axis of length 1
    for tk, tv in ((k[:, :, :1].contiguous(), v), (v.clone(), v.as_strided(v.shape, (999, *v.stride()[1:2], 7, *v.stride()[3:])))):
        _check_attend(_rows(g, 1, 3, 2, HD).cuda(), cache, tk, tv)
    from vitxt_gqa_amd import decode
    with pytest.raises(ValueError, match="same strides"):
        decode.attend(_rows(g, 1, 3, 2, HD).cuda(), cache, v, wide)


def test_attend_peaky_scores():
    """Scores of hundreds of nats, rising and falling along the cache: the running maximum moves at every block, late and early ones dominate."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(23)
    L = 900
    for ramp in (torch.linspace(-1, 1, L), torch.linspace(1, -1, L), torch.where(torch.arange(L) == 517, 1.0, -1.0)):
        k = _rows(g, 1, L, 1, HD) * 0.01
        k[0, :, 0, 0] = ramp * 12
        v = _rows(g, 1, L, 1, HD)
        cache = decode.KVCache8(1, 1, L, "int8")
        cache.append(k.cuda(), v.cuda())
        for top in (-220.0, -30.0, 0.0, 30.0, 220.0):
            q = torch.zeros(1, 2, 1, HD)
            q[0, 0, 0, 0] = top
            q[0, 1] = _rows(g, 1, HD)
            for dt in (torch.float32, torch.bfloat16):
                _check_attend(q.to(dt).cuda(), cache)
    _check_attend(torch.zeros(1, 1, 1, HD).cuda(), cache, scale=1.0)
    _check_attend(_rows(g, 1, 1, 1, HD).cuda(), cache, scale=-0.3)


def test_attend_stale_codes_behind_the_length():
    """Blocks cut back by set_lens, and NaN codes (e4m3 0x7f) and NaN scales behind a sequence's length, change nothing."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(24)
    cache = _filled(g, 2, 2, [200, 200], "e4m3", cap=256)
    q = _rows(g, 2, 2, 2, HD).cuda()
    for n in ([70, 1], [64, 65], [0, 128]):
        cache.set_lens(torch.tensor(n, dtype=torch.int32).cuda())
        got = _check_attend(q, cache)
        kc, vc, ks, vs = cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone()
        kb, vb = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
        from decode_ref import ORDER
        at = torch.tensor(ORDER, device="cuda")
        for b in range(2):
            full, part = divmod(n[b], BLOCK)
            kb[b, :, full, part:] = 0x7f
            vb[b, :, full][..., at >= part] = 0x7f
            kb[b, :, full + 1:], vb[b, :, full + 1:] = 0x7f, 0xff
            cache.k_scale[b, :, -(-n[b] // BLOCK):] = math.nan
            cache.v_scale[b, :, -(-n[b] // BLOCK):] = math.inf
        again = decode.attend(q, cache)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
        kk, vv = cache.dequantize(torch.float32)
        assert not torch.isnan(kk).any() and not torch.isnan(vv).any()
        cache.k.copy_(kc), cache.v.copy_(vc), cache.k_scale.copy_(ks), cache.v_scale.copy_(vs)


def test_attend_any_bound_any_share():
    """max_len only shapes the launch: too small, too large and exact bounds give right results; a call repeats bit for bit."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(25)
    cache = _filled(g, 2, 1, [1900, 300], "int8", cap=4096)
    q = _rows(g, 2, 3, 1, HD, dtype=torch.bfloat16).cuda()
    for bound in (0, 1, 300, 1900, 4096):
        cache.max_len = bound
        a = _check_attend(q, cache)
        b = decode.attend(q, cache)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    cache.lens[0] = 5000                                                                       # a length that cannot be: NaN, nothing is read
    out, lse = decode.attend(q, cache)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and not torch.isnan(out[1]).any()


def test_attend_offsets_beyond_32_bits():
    """2^26 + 100 tokens of one head: 4.3 GB of keys and as much of values; the last block decides, then a token is appended behind it."""
    from vitxt_gqa_amd import decode
    L = (1 << 26) + 100
    n = -(-(L + 1) // BLOCK)
    k, v = (torch.zeros(1, 1, n, BLOCK, HD, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(1, 1, n, device="cuda") for _ in range(2))
    cache = decode.KVCache8.from_parts(k, v, ks, vs, torch.tensor([L], dtype=torch.int32, device="cuda"))
    from decode_ref import ORDER
    last = L - 1
    blk, tok = divmod(last, BLOCK)
    k[0, 0, blk, tok, 0] = 100
    v[0, 0, blk, :, ORDER.index(tok)] = torch.arange(HD, device="cuda", dtype=torch.int8)
    q = torch.zeros(1, 1, 1, HD, device="cuda")
    q[..., 0] = 2.4                                                                            # score 30: e^30 against 2^26
    out, lse = decode.attend(q, cache)
    s = 0.125 * 100 * float(q[0, 0, 0, 0])
    w = math.exp(s) / (math.exp(s) + L - 1)
    assert abs(float(lse) - math.log(math.exp(s) + L - 1)) <= 200 * U * s + (L / 32 / 256 + 64) * U + U * s
    assert bool(((out.flatten().cpu() - w * torch.arange(64)).abs() <= (400 * U * s + 1e-4) * 63).all())
    x = torch.full((1, 1, 1, HD), 3.0, device="cuda")
    cache.append(x, -x)
    assert cache.lens.tolist() == [L + 1]
    blk, tok = divmod(L, BLOCK)
    assert float(cache.k_scale[0, 0, blk]) * int(k[0, 0, blk, tok, 9]) == pytest.approx(3.0) and float(cache.v_scale[0, 0, blk]) * int(v[0, 0, blk, 9, ORDER.index(tok)]) == pytest.approx(-3.0, rel=0.2)


# ---- selection -------------------------------------------------------------------------------------------------------------------------------
def _check_select(logits, scores, K, finished=None, pad=0):
    from vitxt_gqa_amd import decode
    dev = lambda t: None if t is None else t.cuda()
    got, parents, tokens = decode.beam_select(dev(logits), dev(scores), K, dev(finished), pad)
    best, rp, rt = select_ref(logits, scores, K, finished, pad)
    got, parents, tokens, ref = got.cpu().double(), parents.cpu(), tokens.cpu(), best[:, :K]
    inf = ref == -math.inf
    assert torch.equal(got == -math.inf, inf)
    tol = 160 * U + U * ref.abs()
    assert bool(((got - ref).abs() <= tol)[~inf].all()), "score off by %.3g" % (got - ref)[~inf].abs().max()
    # wherever a rank is not within the tolerance of a neighbour's score, without being equal to it, the candidate is the statement's
    gap = torch.full((ref.shape[0], K), math.inf, dtype=torch.float64)
    step = best[:, :-1] - best[:, 1:]
    step = torch.where(torch.isnan(step) | (step == 0), torch.full_like(step, math.inf), step)
    n = step.shape[1]
    gap[:, :n] = torch.minimum(gap[:, :n], step[:, :K])
    gap[:, 1:] = torch.minimum(gap[:, 1:], step[:, :K - 1])
    clear = gap > 2 * (160 * U)
    assert torch.equal(parents[clear], rp[clear]) and torch.equal(tokens[clear], rt[clear])
    assert float(clear.double().mean()) > 0.9
    return got, parents, tokens


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,N,V,K", [(1, 1, 1, 1), (2, 3, 1, 3), (3, 1, 50, 5), (2, 5, 5600, 5), (1, 4, 4095, 8), (1, 4, 4096, 8), (1, 4, 4097, 8), (5, 2, 300, 32), (2, 32, 999, 32), (1, 13, 30522, 26),
                                     (1, 2, 140001, 7), (1, 1, 270000, 32), (40, 8, 1024, 16)])
def test_select(dtype, B, N, V, K):
    g = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(B, N, V, generator=g) * 2).to(DT[dtype])
    scores = -torch.rand(B, N, generator=g) * 6
    _check_select(logits, scores, K)
    fin = torch.rand(B, N, generator=g) < 0.4
    _check_select(logits.masked_fill(torch.rand(B, N, V, generator=g) < 0.5, -math.inf), scores, K, fin, pad=V // 2)


def test_select_ties_go_to_the_lowest_index():
    g = torch.Generator().manual_seed(31)
    V, N, K = 9000, 4, 16
    _, p, t = _check_select(torch.zeros(2, N, V), torch.zeros(2, N), K)                       # everything equal
    assert p.eq(0).all() and torch.equal(t, torch.arange(K).expand(2, K))
    row = torch.randint(0, 3, (V,), generator=g).float()                                      # three values, the same row in every beam
    _check_select(row.expand(2, N, V).contiguous(), torch.zeros(2, N), K)
    _check_select(row.expand(1, N, V).contiguous(), torch.tensor([[-1.0, 0.0, 0.0, -1.0]]), K)
    z = torch.zeros(1, 1, 70)
    z[0, 0, ::2] = -0.0                                                                        # -0 and 0 are one number
    _, _, t = _check_select(z, torch.zeros(1, 1), 5)
    assert t.tolist() == [[0, 1, 2, 3, 4]]


def test_select_negative_zeros_on_top():
    """Rows whose best logits are -0.0: the same number as 0, and not below a bound of it."""
    for V in (4096, 9001):
        for dtype in (torch.float32, torch.bfloat16):
            x = torch.full((2, 2, V), -3.0, dtype=dtype)
            x[:, :, 5::16] = -0.0
            _, _, t = _check_select(x, torch.tensor([[0.0, -9.0]] * 2), 7)
            assert t.tolist() == [list(range(5, 5 + 7 * 16, 16))] * 2
            _, _, t = _check_select(torch.full((1, 1, V), -0.0, dtype=dtype), torch.zeros(1, 1), 32)
            assert t.tolist() == [list(range(32))]


@pytest.mark.parametrize("order", ["up", "down", "lanes", "stretches", "few", "steps"])
def test_select_in_orders_that_defeat_the_bound(order):
    """Orders in which a lane's or a wave's best says little of the others: rising, falling, the best in one lane, in one stretch, almost all masked, few values."""
    g = torch.Generator().manual_seed(36)
    for V, N, K in ((4096, 2, 32), (9000, 3, 32), (30000, 2, 5), (70001, 1, 32)):
        x = torch.sort(torch.randn(2, N, V, generator=g) * 3, -1).values
        at = torch.arange(V)
        if order == "down":
            x = x.flip(-1)
        elif order == "lanes":                                  # the largest logits 1 024 elements apart
            to = torch.argsort(at % 1024, stable=True)
            x = torch.empty_like(x).index_copy_(2, to, x.flip(-1))
        elif order == "stretches":
            x = x.roll(V // 2 + 17, -1)
        elif order == "few":
            x = torch.where(torch.rand(2, N, V, generator=g) < 20.0 / V, x, torch.full_like(x, -math.inf))
        elif order == "steps":
            x = (x * 2).round() / 2
        s = -torch.rand(2, N, generator=g)
        for dt in (torch.float32, torch.bfloat16):
            _check_select_ordered(x.to(dt), s, K)
            _check_select_ordered(x.to(dt), torch.zeros(2, N), K)


def _check_select_ordered(x, s, K, finished=None, pad=0):
    """The statement's order wherever its scores differ clearly; equal logits of a row in the order of their places."""
    from vitxt_gqa_amd import decode
    got, p, t = (r.cpu() for r in decode.beam_select(x.cuda(), s.cuda(), K, None if finished is None else finished.cuda(), pad))
    best, rp, rt = select_ref(x, s, K, finished, pad)
    ref = best[:, :K]
    inf = ref == -math.inf
    assert torch.equal(got.double() == -math.inf, inf) and bool(((got.double() - ref).abs() <= 160 * U + U * ref.abs())[~inf].all())
    V, N = x.shape[2], x.shape[1]
    full = select_ref(x, s, N * V, finished, pad)                                  # every candidate's score, at its place
    total = torch.empty_like(full[0]).scatter_(1, full[1] * V + full[2], full[0])
    for b in range(x.shape[0]):
        picked = (p[b] * V + t[b]).tolist()
        assert len(set(picked)) == K and all(0 <= w < V for w in t[b].tolist()) and all(0 <= n < N for n in p[b].tolist())
        mine = total[b, picked]
        assert torch.equal(mine == -math.inf, inf[b])
        assert bool(((mine - ref[b])[~inf[b]].abs() <= 2 * 160 * U).all())         # a permutation among scores that are equal up to the tolerance at most
        for i in range(1, K):
            # (beside an infinite logit, which counts as 3.4e38, every x - 3.4e38 is -3.4e38 in 64 bits: not a tie of the logits)
            if p[b, i] == p[b, i - 1] and mine[i] == mine[i - 1] and x[b, p[b, i]].max() < math.inf:
                assert t[b, i] > t[b, i - 1]
        assert picked[int((~inf[b]).sum()):] == (rp[b] * V + rt[b]).tolist()[int((~inf[b]).sum()):]      # at -inf: the lowest places


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,V", [(32, 1), (1, 33), (32, 1024), (31, 1024), (16, 2048), (1, 32768), (4, 8192), (5, 6144), (3, 10241), (8, 4097), (13, 63), (2, 16384), (2, 16385), (32, 1025)])
def test_select_few_logits(dtype, N, V):
    """Sequences on either side of what one workgroup holds: all beams alike, one beam, masked, tied, ended, in falling order, hardly a number left."""
    g = torch.Generator().manual_seed(38 + N + V)
    x = (torch.randn(3, N, V, generator=g) * 2).to(DT[dtype])
    s = -torch.rand(3, N, generator=g) * 6
    fin = torch.rand(3, N, generator=g) < 0.4
    first = torch.full((3, N), -math.inf)
    first[:, 0] = 0.0
    apart = -torch.arange(N).float().expand(3, N) * 7                                           # one beam far ahead of the others
    for K in sorted({1, min(5, N * V), min(N, N * V), min(32, N * V)}):
        _check_select_ordered(x, s, K)
        _check_select_ordered(x, s, K, fin, V - 1)
        _check_select_ordered(x, first, K)
        _check_select_ordered(x, apart, K)
        _check_select_ordered(x, apart.flip(1), K, fin, V // 3)
        _check_select_ordered(x, torch.zeros(3, N), K, torch.ones(3, N, dtype=torch.bool), V // 2)
        _check_select_ordered(x.masked_fill(torch.rand(3, N, V, generator=g) < 0.97, -math.inf), s, K, fin, 0)
        _check_select_ordered(torch.zeros_like(x), torch.zeros(3, N), K)
        _check_select_ordered((x / 2).round(), s, K)
        _check_select_ordered(torch.sort(x, -1, descending=True).values, s, K)
        _check_select_ordered(x.masked_fill(torch.rand(3, N, V, generator=g) < 0.5, torch.finfo(DT[dtype]).min), s, K)
        comb = x + 40 * (torch.arange(V) % 64 < 33).to(x.dtype)                                 # the best logits of a wave in few lanes
        _check_select_ordered(comb, s, K)
        _check_select_ordered((comb / 16).round(), s, K, fin, V // 2)
        bad = x.clone()
        bad[0, 0, V // 3], bad[1, N - 1, V - 1], bad[2, N // 2, 0] = math.nan, math.inf, math.nan
        _check_select_ordered(bad, s, K)


def test_select_rows_that_start_anywhere():
    """Many rows (several stretches to a workgroup) and lengths around a stretch, at every offset of a 16-byte unit."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(37)
    for B, N, V in ((1, 3, 4090), (1, 3, 4093), (300, 8, 8189), (70, 32, 4095)):
        wide = (torch.randn(B, N, V + 9, generator=g) * 2)
        s = -torch.rand(B, N, generator=g) * 4
        for dt, step in ((torch.float32, 4), (torch.bfloat16, 8)):
            w = wide.to(dt).cuda()
            for at in range(0, step, 1 if B == 1 else 3):
                view = w[:, :, at:at + V]
                a, b = decode.beam_select(view, s.cuda(), N), decode.beam_select(view.contiguous(), s.cuda(), N)
                assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2]) and bool(((a[0] - b[0]).abs() <= 2 * 160 * U + U * b[0].abs()).all())
            if B == 1:
                _check_select(w[:, :, 1:1 + V].cpu().contiguous(), s, N)


def test_select_first_step_and_dead_beams():
    g = torch.Generator().manual_seed(32)
    logits = torch.randn(2, 5, 700, generator=g)
    scores = torch.full((2, 5), -math.inf)
    scores[:, 0] = 0.0
    _, p, _ = _check_select(logits, scores, 5)
    assert p.eq(0).all()
    _, p, t = _check_select(logits, torch.full((2, 5), -math.inf), 7)                         # nothing at all: the lowest candidates, at -inf
    assert p.eq(0).all() and torch.equal(t, torch.arange(7).expand(2, 7))
    scores[1, 2] = math.nan
    _check_select(logits, scores, 5)


def test_select_masked_and_not_finite():
    g = torch.Generator().manual_seed(33)
    x = torch.randn(3, 3, 500, generator=g)
    x[0, 0] = -math.inf                                                                        # a row without a word left
    x[0, 1, 10:] = -math.inf
    x[1, 0, 7] = math.nan
    x[1, 1] = math.nan
    x[1, 2, 100:] = torch.finfo(torch.float32).min                                             # masks of the type's lowest value
    x[2] = -math.inf                                                                           # a sequence without any
    _check_select(x, torch.zeros(3, 3), 12)
    _check_select(x[:, :, :3].contiguous(), torch.zeros(3, 3), 9)
    low = torch.full((1, 2, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    low[0, 1, 5] = 1.0
    _check_select(low, torch.zeros(1, 2), 4)
    big = torch.zeros(1, 2, 300)
    big[0, 0, 9] = math.inf
    got, p, t = _check_select(big, torch.zeros(1, 2), 1)
    assert (float(got), int(p), int(t)) == (0.0, 0, 9)


def test_select_finished():
    g = torch.Generator().manual_seed(34)
    x = torch.randn(2, 4, 9000, generator=g)
    s = -torch.rand(2, 4, generator=g)
    _check_select(x, s, 6, torch.ones(2, 4, dtype=torch.bool), pad=8999)                       # all ended: four candidates, then the lowest at -inf
    s[0, 2] = -math.inf                                                                        # an ended beam that is none
    x[0, 1] = math.nan                                                                         # logits of an ended beam are not read
    f = torch.tensor([[False, True, True, False], [False] * 4])
    for pad in (0, 5, 4096, 8999):
        got, p, t = _check_select(x, s, 8, f, pad)
        assert not torch.isnan(got).any()
    _check_select(x, s, 8, f.to(torch.uint8), 3)
    _check_select(x[:, :, :6].contiguous(), s, 24, f, 3)                                        # every candidate there is


def test_select_views():
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(35)
    wide = torch.randn(3, 12, 2001, generator=g).cuda()
    view = wide[:, 2:10:2, 1:1990]                                                             # odd row stride, rows that start anywhere
    s = (-torch.rand(4, 3, generator=g)).t()
    a = decode.beam_select(view, s.cuda().contiguous(), 4)
    b = decode.beam_select(view.contiguous(), s.cuda().t().contiguous().t(), 4)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    _check_select(view.cpu().contiguous(), s.contiguous(), 4)
    one = wide[:, :1, :500].expand(-1, 4, -1)                                                  # one row for every beam
    _check_select(one.cpu().contiguous(), s.contiguous(), 4)
    assert torch.equal(decode.beam_select(one, s.cuda(), 4)[2], decode.beam_select(one.contiguous(), s.cuda(), 4)[2])
    out = decode.beam_select(wide[:0], torch.zeros(0, 12, device="cuda"), 3)
    assert [tuple(x.shape) for x in out] == [(0, 3)] * 3


# ---- reordering ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,d,dtype", [((3, 5), 0, torch.int64), ((2, 3, 5, 12, 64), 1, torch.bfloat16), ((2, 2, 32, 7), 1, torch.uint8), ((4, 1, 9), 0, torch.float32), ((4, 13, 3, 3), 0, torch.bfloat16),
                                           ((6, 16, 1, 5), 0, torch.int32), ((2, 3, 2, 4, 31, 3), 2, torch.float64), ((1, 4, 1024, 33), 0, torch.float32), ((2, 8, 11), 0, torch.bool)])
def test_reorder(shape, d, dtype):
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(len(shape))
    x = torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=g).to(dtype)
    B, N = shape[d], shape[d + 1]
    flat = x.reshape(-1, B, N, *shape[d + 2:])
    kinds = [torch.randint(0, N, (B, N), generator=g), torch.arange(N).expand(B, N), torch.zeros(B, N, dtype=torch.int64), torch.arange(N).flip(0).expand(B, N), torch.randint(-3, N + 3, (B, N), generator=g)]
    for parents in kinds:
        for used in [None] + ([0, 1, shape[d + 2]] if len(shape) > d + 2 else []):
            want = flat.clone()
            for b in range(B):
                for n in range(N):
                    p = min(max(int(parents[b, n]), 0), N - 1)
                    if used is None:
                        want[:, b, n] = flat[:, b, p]
                    else:
                        want[:, b, n, :used] = flat[:, b, p, :used]
            y = x.clone().cuda()
            assert decode.beam_reorder(y, parents.cuda(), batch_dim=d, used=used) is y
            assert torch.equal(y.cpu(), want.reshape(shape)), (parents, used)
    assert decode.beam_reorder(torch.zeros(0, 3, 4).cuda(), torch.zeros(0, 3, dtype=torch.int64).cuda()).shape == (0, 3, 4)


# ---- refusals --------------------------------------------------------------------------------------------------------------------------------
def test_gradients_are_refused():
    from vitxt_gqa_amd import decode
    cache = decode.KVCache8(1, 1, 64)
    x = torch.zeros(1, 1, 1, HD, device="cuda", requires_grad=True)
    for call in (lambda: cache.append(x, x), lambda: decode.attend(x, cache), lambda: decode.beam_select(torch.zeros(1, 1, 5, device="cuda", requires_grad=True), torch.zeros(1, 1, device="cuda"), 1),
                 lambda: decode.beam_reorder(torch.zeros(1, 2, 5, device="cuda", requires_grad=True), torch.zeros(1, 2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError, match="no gradients"):
            call()
    with torch.no_grad():
        decode.attend(x, cache)
    with pytest.raises(ValueError, match="one device"):
        decode.attend(torch.zeros(1, 1, 1, HD), cache)
