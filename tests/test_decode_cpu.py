"""The decode operators' refusals (no kernel is launched) and the plain statements they are tested against."""
import ctypes

import pytest
import torch

from decode_ref import RefCache, round_e4m3, scale_of, select_ref
from vitxt_gqa_amd import decode, hipext


@pytest.fixture(scope="module")
def lib():
    from vitxt_gqa_amd import build
    build.build(verbose=False)
    return hipext.lib()


def _cache(B=2, H=3, cap=100, fmt="int8"):
    return decode.KVCache8(B, H, cap, fmt, device="cpu")


def test_cache_shapes():
    c = _cache()
    assert c.capacity == 128 and c.blocks == 2 and c.k.shape == (2, 3, 2, 64, 64) and c.k.dtype == torch.int8 and c.v.shape == c.k.shape
    assert c.k_scale.shape == (2, 3, 2) and c.lens.tolist() == [0, 0]
    assert _cache(fmt="e4m3").k.dtype == torch.float8_e4m3fn
    d = decode.KVCache8.from_parts(c.k, c.v, c.k_scale, c.v_scale, c.lens)
    assert d.k.data_ptr() == c.k.data_ptr() and d.fmt == "int8" and d.max_len == 128
    assert c.set_lens(7).lens.tolist() == [7, 7] and c.max_len == 7
    assert c.set_lens(torch.tensor([3, 9], dtype=torch.int32)).lens.tolist() == [3, 9]


def test_cache_storage_is_its_own():
    """The storage of a cache stays what it was made with; copies have addresses of their own."""
    import copy
    import io
    c = _cache().set_lens(5)
    with pytest.raises(AttributeError):
        c.k = torch.zeros_like(c.k)
    with pytest.raises(AttributeError):
        c.lens = torch.zeros_like(c.lens)
    buf = io.BytesIO()
    torch.save(c, buf)
    buf.seek(0)
    for d, own in ((copy.deepcopy(c), True), (torch.load(buf, weights_only=False), True), (copy.copy(c), False)):
        assert d._ptrs == tuple(t.data_ptr() for t in (d.k, d.v, d.k_scale, d.v_scale, d.lens)) and d._ticket_ptr == d._ticket.data_ptr() != c._ticket_ptr
        assert (d.k.data_ptr() != c.k.data_ptr()) == own and d.lens.tolist() == [5, 5] and (d.max_len, d.fmt, d.capacity) == (5, "int8", 128)
    assert decode.KVCache8.from_parts(c.k, c.v, c.k_scale, c.v_scale, c.lens, -3).max_len == 0


@pytest.mark.parametrize("make", [
    lambda c: decode.KVCache8(2, 3, 64, "int4", device="cpu"),
    lambda c: decode.KVCache8(0, 3, 64, device="cpu"),
    lambda c: decode.KVCache8(2, 3, 0, device="cpu"),
    lambda c: decode.KVCache8.from_parts(c.k, c.v.view(torch.float8_e4m3fn), c.k_scale, c.v_scale, c.lens),
    lambda c: decode.KVCache8.from_parts(c.k[:, :, :, :, :32], c.v, c.k_scale, c.v_scale, c.lens),
    lambda c: decode.KVCache8.from_parts(c.k.transpose(0, 1), c.v.transpose(0, 1), c.k_scale.transpose(0, 1), c.v_scale.transpose(0, 1), c.lens),
    lambda c: decode.KVCache8.from_parts(c.k, c.v, c.k_scale.double(), c.v_scale, c.lens),
    lambda c: decode.KVCache8.from_parts(c.k, c.v, c.k_scale, c.v_scale, c.lens.long()),
    lambda c: c.set_lens(129),
    lambda c: c.set_lens(-1),
    lambda c: c.set_lens(torch.zeros(2, dtype=torch.int64)),
    lambda c: c.dequantize(torch.float16),
    lambda c: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64, dtype=torch.bfloat16)),
    lambda c: c.append(torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 4, 64)),
    lambda c: c.append(torch.zeros(3, 5, 3, 64), torch.zeros(3, 5, 3, 64)),
    lambda c: c.append(torch.zeros(2, 5, 3, 32), torch.zeros(2, 5, 3, 32)),
    lambda c: c.append(torch.zeros(2, 5, 3, 64, dtype=torch.float16), torch.zeros(2, 5, 3, 64, dtype=torch.float16)),
    lambda c: c.append(torch.zeros(2, 129, 3, 64), torch.zeros(2, 129, 3, 64)),
    lambda c: c.append(torch.zeros(2, 5, 3, 65)[..., 1:], torch.zeros(2, 5, 3, 65)[..., 1:]),
    lambda c: c.append(torch.zeros(2, 5, 64, 3).transpose(2, 3), torch.zeros(2, 5, 64, 3).transpose(2, 3)),
    lambda c: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64), counts=torch.zeros(2, dtype=torch.int64)),
    lambda c: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64), counts=torch.zeros(3, dtype=torch.int32)),
    lambda c: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64), rows=torch.zeros(2, 5, dtype=torch.int64)),
    lambda c: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64), rows=torch.zeros(5, 2, dtype=torch.int32).t()),
    lambda c: c.append(torch.zeros(2, 0, 3, 64), torch.zeros(2, 0, 3, 64), rows=torch.zeros(2, 5, dtype=torch.int32)),
    lambda c: decode.attend(torch.zeros(2, 1, 4, 64), c),
    lambda c: decode.attend(torch.zeros(3, 1, 3, 64), c),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 128), c),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64, dtype=torch.float16), c),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 66)[..., 2:], c),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 1, 4, 3, 64)),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 2, 4, 3, 64), torch.zeros(2, 2, 4, 3, 64)),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64)),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 1, 4, 3, 64).bfloat16(), torch.zeros(2, 1, 4, 3, 64).bfloat16()),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 1, 4, 3, 64), torch.zeros(2, 1, 3, 4, 64).transpose(2, 3)),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, torch.zeros(2, 1, 4, 3, 64), torch.zeros(2, 1, 4, 3, 64), torch.zeros(2, 1, dtype=torch.int64)),
    lambda c: decode.attend(torch.zeros(2, 1, 3, 64), c, tail_len=3),
])
def test_cache_and_attention_refuse(make):
    with pytest.raises(ValueError):
        make(_cache())


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(2, 3)), dict(logits=torch.zeros(2, 3, 0)), dict(logits=torch.zeros(2, 3, 5).half()), dict(logits=torch.zeros(2, 5, 3).transpose(1, 2)),
    dict(scores=torch.zeros(2, 2)), dict(scores=torch.zeros(2, 3).double()), dict(n_select=0), dict(n_select=33), dict(n_select=16), dict(pad=-1), dict(pad=5),
    dict(finished=torch.zeros(2, 3)), dict(finished=torch.zeros(3, 2, dtype=torch.bool)), dict(logits=torch.zeros(2, 33, 5), scores=torch.zeros(2, 33))])
def test_select_refuses(kw):
    with pytest.raises(ValueError):
        decode.beam_select(**{**dict(logits=torch.zeros(2, 3, 5), scores=torch.zeros(2, 3), n_select=3), **kw})


@pytest.mark.parametrize("kw", [
    dict(state=torch.zeros(2, 4, 3).transpose(1, 2)), dict(parents=torch.zeros(2, 3, dtype=torch.int32)), dict(parents=torch.zeros(3, 2, dtype=torch.int64)), dict(used=5), dict(used=-1),
    dict(batch_dim=2), dict(batch_dim=-4), dict(state=torch.zeros(2, 33, 4), parents=torch.zeros(2, 33, dtype=torch.int64)),
    dict(state=torch.zeros(2, 3), used=1)])
def test_reorder_refuses(kw):
    with pytest.raises(ValueError):
        decode.beam_reorder(**{**dict(state=torch.zeros(2, 3, 4), parents=torch.zeros(2, 3, dtype=torch.int64)), **kw})


def test_no_cpu_path():
    c = _cache()
    for call in (lambda: c.append(torch.zeros(2, 5, 3, 64), torch.zeros(2, 5, 3, 64)), lambda: c.dequantize(), lambda: decode.attend(torch.zeros(2, 1, 3, 64), c),
                 lambda: decode.beam_select(torch.zeros(2, 3, 5), torch.zeros(2, 3), 3), lambda: decode.beam_reorder(torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_c_abi_refuses(lib):
    p = ctypes.c_void_p(16)
    ok = [p, 0, 64, 64, p, 0, 64, 64, None, 0, None, p, p, p, p, p, p, 1, 1, 1, 1, 1, 0, 0, None]

    def append(**at):
        a = list(ok)
        for i, v in at.items():
            a[int(i[1:])] = v
        return lib.t2s_kv8_append(*a), lib.t2s_last_error()

    for kw, text in ((dict(_0=None), b"null pointer"), (dict(_17=0), b"bad shape"), (dict(_19=2), b"tokens of"), (dict(_22=7), b"bad dtype"), (dict(_23=2), b"bad format"),
                     (dict(_2=62), b"aligned"), (dict(_11=ctypes.c_void_p(8)), b"aligned")):
        rc, err = append(**kw)
        assert rc != 0 and text in err, (kw, err)
    assert lib.t2s_kv8_dequantize(p, p, p, p, p, p, ctypes.c_void_p(8), 1, 1, 1, 0, 0, None) != 0 and b"alignment" in lib.t2s_last_error()
    att = [p, 0, 64, 64, p, p, p, p, p, None, None, 0, 0, 0, 0, None, 0, 0, 0, p, p, p, 1 << 20, 2, 1, 1, 1, 1, 1, 0.125, 0, 0, None]
    for i, v, text in ((0, None, b"null pointer"), (24, 0, b"bad shape"), (9, p, b"come together"), (22, 8, b"too small"), (23, 0, b"too small"), (2, 63, b"aligned"), (30, 3, b"bad dtype"), (31, 3, b"bad format")):
        a = list(att)
        a[i] = v
        assert lib.t2s_kv8_attn(*a) != 0 and text in lib.t2s_last_error(), (i, lib.t2s_last_error())
    sel = [p, 40000, 40000, p, None, 0, p, p, p, p, 1 << 20, 1, 3, 40000, 3, 0, None]
    for i, v, text in ((0, None, b"null pointer"), (12, 33, b"bad shape"), (14, 33, b"candidates"), (5, 40000, b"pad"), (10, 8, b"too small"), (15, 2, b"bad dtype")):
        a = list(sel)
        a[i] = v
        assert lib.t2s_beam_select(*a) != 0 and text in lib.t2s_last_error(), (i, lib.t2s_last_error())
    assert lib.t2s_beam_reorder(p, p, 1, 1, 33, 16, 16, None) != 0 and b"bad shape" in lib.t2s_last_error()
    assert lib.t2s_beam_reorder(p, p, 1, 1, 3, 16, 32, None) != 0 and b"bytes" in lib.t2s_last_error()
    assert lib.t2s_kv8_attn_splits(0, 1, 1, 1, 64, 0) == 0 and lib.t2s_kv8_attn_splits(1, 1, 1, 1, 0, 1) == 1
    assert lib.t2s_beam_select_workspace_bytes(0, 1, 1, 1) == 0 == lib.t2s_beam_select_workspace_bytes(1, 5, 5600, 5) < lib.t2s_beam_select_workspace_bytes(1, 3, 40000, 3)
    # shapes whose products pass 32 bits are refused, none ends the process
    big = 2 ** 31 - 1
    assert lib.t2s_kv8_attn_splits(1, 65536, 1, 65536, 64, 0) == 0 and lib.t2s_kv8_attn_splits(big, 1, big, 1, 64, 0) == 0 and lib.t2s_kv8_attn_splits(1, 1, 1, 1, big, 0) > 1
    assert lib.t2s_kv8_attn_workspace_bytes(1, 65536, 1, 65536, 2) == 0 and lib.t2s_kv8_attn_workspace_bytes(1, 1, 1, 1, 0) == 0
    for n, h, grp in ((65536, 1, 65536), (big, big, 1), (4097, 4096, 1)):
        a = list(att)
        a[25], a[26], a[27] = n, h, grp
        assert lib.t2s_kv8_attn(*a) != 0 and b"bad shape" in lib.t2s_last_error()
    a = list(sel)
    a[10:14] = big, 1 << 24, 3, 40000
    assert lib.t2s_beam_select(*a) != 0 and (b"too many rows" in lib.t2s_last_error() or b"too small" in lib.t2s_last_error())
    assert lib.t2s_beam_reorder(p, p, 1, 1, 3, 1 << 40, 1 << 40, None) != 0 and b"too long" in lib.t2s_last_error()


def test_reference_statements():
    """The plain forms themselves: e4m3 rounding against torch's cast, scales, a tie to the lowest index."""
    x = torch.linspace(-448, 448, 20011)
    assert torch.equal(round_e4m3(x), x.to(torch.float8_e4m3fn).double())
    assert torch.equal(round_e4m3(x / 1000), (x / 1000).to(torch.float8_e4m3fn).double())
    assert float(scale_of(torch.tensor(448.0), "e4m3")) == 1.0 and float(scale_of(torch.tensor(448.1), "e4m3")) == 2.0 and float(scale_of(torch.tensor(0.0), "e4m3")) > 0
    assert float(scale_of(torch.tensor(127.0), "int8")) == 1.0
    r = RefCache(1, 1, "int8")
    r.append(torch.ones(1, 65, 1, 64), torch.ones(1, 65, 1, 64))
    assert r.lens() == [65] and len(r.scales[0][0][0]) == 2 and (r.values(0, 0, 0) - 1).abs().max() < 1e-6
    s, p, t = select_ref(torch.zeros(1, 2, 3), torch.zeros(1, 2), 4)
    assert p.tolist() == [[0, 0, 0, 1]] and t.tolist() == [[0, 1, 2, 0]]
