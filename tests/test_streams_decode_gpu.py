"""The decode operators (vitxt_gqa_amd/decode.py) on streams, in threads and in captured graphs.  In a file of their own behind the other tests that use
streams: streams come from a pool in turn and share a few hardware queues, and test_handoff_guard_gpu.py needs two that do not."""
import pytest
import torch

from test_decode_gpu import HD, _filled, _rows

pytestmark = pytest.mark.gpu


def test_on_another_stream():
    """The calls run on the current stream, behind what it holds."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(41)
    k, v, q = _rows(g, 2, 3000, 2, HD).cuda(), _rows(g, 2, 3000, 2, HD).cuda(), _rows(g, 2, 2, 2, HD).cuda()
    logits, s, par = torch.randn(2, 3, 50000, generator=g).cuda(), torch.zeros(2, 3).cuda(), torch.tensor([[2, 0, 0], [1, 2, 0]]).cuda()
    st0 = torch.randn(2, 3, 4096, generator=g).cuda()

    def work():
        cache = decode.KVCache8(2, 2, 3000)
        slow = (torch.ones(2048, 2048, device="cuda") @ torch.ones(2048, 2048, device="cuda"))[0, 0] * 0          # what the stream is busy with
        cache.append(k + slow, v + slow)
        state = st0.clone()
        return (*decode.attend(q + slow, cache), *decode.beam_select(logits + slow, s, 3), decode.beam_reorder(state, par), *cache.dequantize())

    want = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_captured_step_replays():
    """One decode step (append, attend, select, reorder) captured once and replayed over a growing cache, eager work in between, beside a second graph on the
    same cache; every replay equals the eager step."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(42)
    B, H, N, V = 2, 2, 3, 5000
    steps = [[t.cuda() for t in (_rows(g, B, 1, H, HD), _rows(g, B, 1, H, HD), _rows(g, B, N, H, HD), torch.randn(B, N, V, generator=g))] for _ in range(70)]
    base = [_rows(g, B, 50, H, HD).cuda() for _ in range(2)]
    cum, state0 = torch.zeros(B, N).cuda(), torch.randint(0, 99, (B, N, 12), generator=g).cuda()

    def step(cache, x, state):
        cache.append(x[0], x[1])
        out, lse = decode.attend(x[2], cache)
        s, p, t = decode.beam_select(x[3], cum, N)
        decode.beam_reorder(state, p)
        return out, lse, s, p, t

    eager, estate = decode.KVCache8(B, H, 192), state0.clone()
    eager.append(*base)
    want = []
    for x in steps:
        want.append([t.clone() for t in step(eager, x, estate)] + [estate.clone()])
    cache, state, buf = decode.KVCache8(B, H, 192), state0.clone(), [t.clone() for t in steps[0]]
    cache.append(*base)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):                                                            # warm up on the side, then take it back
        step(cache, buf, state)
    torch.cuda.current_stream().wait_stream(stream)
    cache.set_lens(0)
    cache.append(*base)
    state.copy_(state0)
    graph, look = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, buf, state)
    with torch.cuda.graph(look):
        kk, vv = cache.dequantize(torch.float32)
    cache.set_lens(0)
    cache.append(*base)
    state.copy_(state0)
    for i, x in enumerate(steps):
        for b, t in zip(buf, x):
            b.copy_(t)
        graph.replay()
        look.replay()
        noise = decode.attend(x[2], cache)                                                     # eager work between the replays
        torch.cuda.synchronize()
        for a, b in zip((*got, state), want[i]):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6) if a.dtype == torch.float32 else torch.equal(a, b), i
        assert torch.equal(noise[0], got[0]) or torch.allclose(noise[0], got[0], rtol=1e-5, atol=1e-6)
        assert cache.lens.tolist() == [51 + i] * B
    for a, b in zip((kk, vv), eager.dequantize(torch.float32)):
        assert torch.equal(a, b)


def test_threads_on_streams_of_their_own():
    """Two threads, each with a stream, a cache and beams of its own, at the same time: what each gets alone."""
    import threading
    from vitxt_gqa_amd import decode

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        L, N = 900 + 700 * seed, 2 + seed
        return [t.cuda() for t in (_rows(g, 3, L, 2, HD), _rows(g, 3, L, 2, HD), _rows(g, 3, N, 4, HD), torch.randn(3, N, 9000 + seed, generator=g), -torch.rand(3, N, generator=g), torch.randn(3, N, 500, generator=g))]

    def work(x, rounds):
        out = []
        for _ in range(rounds):
            cache = decode.KVCache8(3, 2, x[0].shape[1], "int8")
            cache.append(x[0][:, :333], x[1][:, :333]).append(x[0][:, 333:], x[1][:, 333:])
            state = x[5].clone()
            s, p, t = decode.beam_select(x[3], x[4], x[4].shape[1])
            out.append((*decode.attend(x[2], cache), s, p, t, decode.beam_reorder(state, p), cache.lens.clone()))
        return out

    data = [inputs(0), inputs(1)]
    want = [work(x, 1)[0] for x in data]
    torch.cuda.synchronize()
    got, go = [None, None], threading.Barrier(2)

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            go.wait()
            got[i] = work(data[i], 25)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert got[i] is not None and len(got[i]) == 25
        for res in got[i]:
            for a, b in zip(res, want[i]):
                assert torch.equal(a, b)


def test_two_graphs_of_one_pool():
    """Two captured graphs whose workspaces come from one pool, replayed in turn with eager calls between: each replay gives what its inputs give."""
    from vitxt_gqa_amd import decode
    g = torch.Generator().manual_seed(43)
    caches = [_filled(g, 2, 2, [3000, 1234]), _filled(g, 1, 1, [20000], "e4m3")]
    shapes = [((2, 5, 4, HD), (2, 5, 7001)), ((1, 2, 1, HD), (1, 2, 70000))]
    bufs = [(torch.zeros(a).cuda(), torch.zeros(b).cuda(), torch.zeros(b[:2]).cuda()) for a, b in shapes]
    call = lambda i, x: (*decode.attend(x[0], caches[i]), *decode.beam_select(x[1], x[2], 3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            call(i, bufs[i])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.graph(graphs[0]):
        outs.append(call(0, bufs[0]))
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        outs.append(call(1, bufs[1]))
    for turn in range(6):
        for i in ((0, 1), (1, 0), (0, 0), (1, 1), (1, 0), (0, 1))[turn]:
            x = [torch.randn(b.shape, generator=g).cuda() for b in bufs[i]]
            want = call(i, x)
            for b, t in zip(bufs[i], x):
                b.copy_(t)
            graphs[i].replay()
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), (turn, i)
