"""The 8-bit K/V entries and the masked attention as a program uses them: one behind the other on a sequence that grows and is brought back to
its budget, captured into graphs, on other streams, at offsets past 32 bits."""
import numpy as np
import pytest

from kv8_util import State, attention, decode, evict, from_bits, random_state, rounded, to_bits, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,kind,dim,heads,kv_heads", [(0, 30, 128, 8, 2), (1, 1, 64, 4, 4)])
def test_a_conversation_under_a_budget(gpu, code, kind, dim, heads, kv_heads):
    # a prompt in two chunks, decode steps that add up weights, an eviction to 96 positions, more steps, another eviction
    rng = np.random.default_rng(dim)
    budget, sinks, recent, context = 96, 4, 32, 256
    host = State(context, kv_heads, dim, code)
    state, weights = gpu.upload(host.pack()), gpu.buffer(kv_heads * context * 4)
    sums = np.zeros((kv_heads, context), np.float64)
    rule = dict(cap=20.0, window=0)
    length = 0

    def step(rows):
        nonlocal length
        raws = [to_bits(rng.normal(size=(rows, n, dim)).astype(np.float32), kind) for n in (heads, kv_heads, kv_heads)]
        q, k, v = (gpu.upload(r[0]) for r in raws)
        out = gpu.buffer(rows * heads * dim * 2)
        few = rows * (heads // kv_heads) <= 64
        gpu.kv8_write([state], [context], [length], [rows], kv_heads, dim, code, k, v, kind)
        gpu.kv8_attention([state], [context], [length + rows], [rows], heads, kv_heads, dim, code, dim ** -0.5, q, out, kind, cap=20.0,
                          weights=[weights] if few else None)
        got = from_bits(gpu.read(out, np.int16, (rows, heads, dim)), kind)
        host.write(length, raws[1][1].astype(np.float32), raws[2][1].astype(np.float32))
        length += rows
        want, more, size = attention(raws[0][1], *host.values(length), dim ** -0.5, **rule)
        assert np.all(np.abs(got - want) <= tolerance(kind, want, size)), (length, rows)
        if few:
            sums[:, :length] += more
        for b in (q, k, v, out):
            gpu.release(b)

    step(70)
    step(50)
    for phase in range(2):
        for _ in range(20):
            step(1)
        step(5)
        assert gpu.decode_status() == 0
        # the device's own sums decide: the definition is applied to them
        held = gpu.read(weights, np.float32, (kv_heads, context))
        assert np.allclose(held, sums, rtol=1e-4, atol=1e-5)
        target, target_weights, kept = gpu.buffer(gpu.kv8_bytes(context, kv_heads, dim)), gpu.buffer(kv_heads * context * 4), gpu.buffer(kv_heads * budget * 4)
        gpu.kv8_evict([state], [context], [length], [weights], budget, sinks, recent, kv_heads, dim, code, [target], [context], [target_weights], kept)
        moved, at, moved_weights = evict(host, length, held, budget, sinks, recent)
        assert np.array_equal(gpu.read(kept, np.int32, (kv_heads, budget)), at)
        host = State(context, kv_heads, dim, code)
        host.codes[:, :budget], host.scales[:, :budget // 32] = moved.codes, moved.scales
        got = host.unpack(gpu.read(target, np.uint8, (host.pack().size,)))
        assert np.array_equal(decode(got.codes, code), decode(host.codes, code)) and np.array_equal(got.scales, host.scales)
        for b in (state, weights, kept):
            gpu.release(b)
        state, weights, length = target, target_weights, budget
        sums = np.zeros((kv_heads, context), np.float64)
        sums[:, :budget] = moved_weights
    step(1)
    step(40)
    for b in (state, weights):
        gpu.release(b)


class Torch:
    """Inputs of one call of each entry in torch's memory, over an adopted handle."""

    def __init__(self, gpu, seed, length=700, dim=128):
        import torch
        self.torch, self.gpu, self.length, self.dim = torch, gpu, length, dim
        self.heads, self.kv_heads, self.context = 8, 2, rounded(length + 8)
        rng = np.random.default_rng(seed)
        self.host = random_state(rng, self.context, self.kv_heads, dim, 0, length - 1)
        half = lambda *shape: torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to("cuda", torch.bfloat16)  # noqa: E731
        self.state = torch.from_numpy(self.host.pack()).to("cuda")
        self.k, self.v = half(1, self.kv_heads, dim), half(1, self.kv_heads, dim)
        self.q, self.chunk = half(1, self.heads, dim), half(100, self.heads, dim)
        self.dense = [half(300, n, dim) for n in (self.heads, self.kv_heads, self.kv_heads)]
        self.weights = torch.zeros(self.kv_heads, self.context, device="cuda")
        self.target = torch.zeros(gpu.kv8_bytes(512, self.kv_heads, dim), dtype=torch.uint8, device="cuda")
        self.target_weights = torch.zeros(self.kv_heads, 512, device="cuda")
        self.kept = torch.zeros(self.kv_heads, 512, dtype=torch.int32, device="cuda")
        self.outs = [torch.empty_like(x) for x in (self.q, self.chunk, self.dense[0])]

    def run(self):
        g, at = self.gpu, lambda t: t.data_ptr()  # noqa: E731
        one = ([at(self.state)], [self.context])
        g.kv8_write(*one, [self.length - 1], [1], self.kv_heads, self.dim, 0, at(self.k), at(self.v), 30)
        g.kv8_attention(*one, [self.length], [1], self.heads, self.kv_heads, self.dim, 0, 0.1, at(self.q), at(self.outs[0]), 30, weights=[at(self.weights)])
        g.kv8_attention(*one, [self.length], [100], self.heads, self.kv_heads, self.dim, 0, 0.1, at(self.chunk), at(self.outs[1]), 30, window=300)
        g.masked_attention(*(at(x) for x in self.dense), at(self.outs[2]), [120, 180], [120, 180], self.heads, self.kv_heads, self.dim, 30, 0.1)
        g.kv8_evict(*one, [self.length], [at(self.weights)], 500, 4, 100, self.kv_heads, self.dim, 0, [at(self.target)], [512], [at(self.target_weights)],
                    at(self.kept))

    def results(self):
        return [t.cpu() for t in (self.state, self.weights, self.target, self.target_weights, self.kept, *self.outs)]

    def clear(self):
        for t in (self.weights, self.target, self.target_weights, self.kept, *self.outs):
            t.zero_()


def same(a, b):
    return all(bool((x == y).all()) for x, y in zip(a, b))


def test_a_captured_graph_gives_the_eager_bits():
    import torch
    from straydog_b200.backend import Backend
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), Backend.adopt(0, stream.cuda_stream) as gpu:
        a, b = Torch(gpu, 1), Torch(gpu, 2)
        a.run()
        b.run()
        stream.synchronize()
        want = a.results(), b.results()
        graphs = []
        for x in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                x.run()
        # a larger eager call in between: the graphs keep the workspaces they were captured with
        large = Torch(gpu, 3, length=20000)
        large.run()
        for turn in range(3):
            for x in (a, b):
                x.clear()
            for graph in graphs:
                graph.replay()
            large.run()
            stream.synchronize()
            assert same(a.results(), want[0]) and same(b.results(), want[1])
        # other inputs in the same places
        a.q.copy_(b.q)
        a.state.copy_(b.state)
        a.k.copy_(b.k)
        a.v.copy_(b.v)
        a.clear()
        graphs[0].replay()
        stream.synchronize()
        assert same(a.results()[:6], want[1][:6])
        assert gpu.decode_status() == 0
        del graphs


def test_a_workspace_does_not_grow_inside_a_capture():
    import torch
    from straydog_b200.backend import Backend, StraydogError
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), Backend.adopt(0, stream.cuda_stream) as gpu:
        x = Torch(gpu, 1)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(StraydogError, match="capture"):
            with torch.cuda.graph(graph, stream=stream):
                gpu.kv8_attention([x.state.data_ptr()], [x.context], [600], [100], x.heads, x.kv_heads, x.dim, 0, 0.1, x.chunk.data_ptr(), x.outs[1].data_ptr(), 30)
        x.run()
        stream.synchronize()
        first = x.results()
        x.clear()
        x.run()
        stream.synchronize()
        assert same(x.results(), first)


def test_tensors_made_on_another_stream():
    # the inputs are filled by a long chain on one stream; the handle's stream waits for it, not the host
    import torch
    from straydog_b200.backend import Backend
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    with Backend.adopt(0, mine.cuda_stream) as gpu:
        with torch.cuda.stream(mine):
            x = Torch(gpu, 5)
            x.run()
            mine.synchronize()
            want = x.results()
            x.clear()
        keep = x.q.clone(), x.k.clone(), x.state.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            for t in (x.q, x.k, x.state):
                t.zero_()
            busy = torch.ones(4096, 4096, device="cuda")
            for _ in range(20):
                busy = busy @ busy * 1e-4
            for t, value in zip((x.q, x.k, x.state), keep):
                t.copy_(value)
            done = torch.cuda.Event()
            done.record(other)
        mine.wait_event(done)
        x.run()
        mine.synchronize()
        assert same(x.results(), want)


def test_offsets_past_32_bits(gpu):
    # a state of 4.3 GB: the values' plane, the scales and the last rows lie past 2^32 bytes
    rng = np.random.default_rng(3)
    context, dim = 1 << 23, 256
    state = gpu.buffer(gpu.kv8_bytes(context, 1, dim))
    raws = [to_bits(rng.normal(size=(70, n, dim)).astype(np.float32), 1) for n in (4, 1, 1)]
    q, k, v = (gpu.upload(r[0]) for r in raws)
    gpu.kv8_write([state], [context], [context - 70], [70], 1, dim, 0, k, v, 1)
    small = State(128, 1, dim, 0).write(128 - 70, raws[1][1].astype(np.float32), raws[2][1].astype(np.float32))
    out = gpu.buffer(70 * 4 * dim * 2)
    for rows in (1, 8):
        gpu.kv8_attention([state], [context], [context], [rows], 4, 1, dim, 0, dim ** -0.5, q, out, 1, window=60)
        got = from_bits(gpu.read(out, np.int16, (rows, 4, dim)), 1)
        keys, values = small.values(128)
        want, _, size = attention(raws[0][1][:rows], keys, values, dim ** -0.5, window=60)
        assert np.all(np.abs(got - want) <= tolerance(1, want, size)), rows
    assert gpu.decode_status() == 0
    for b in (state, q, k, v, out):
        gpu.release(b)


def test_a_call_twice_has_the_same_bits(gpu):
    rng = np.random.default_rng(4)
    lengths = [3000, 17, 901, 2048]
    states = [random_state(rng, rounded(n), 2, 64, 1, n) for n in lengths]
    buffers = [gpu.upload(s.pack()) for s in states]
    rows = [1, 3, 90, 2]
    q = gpu.upload(to_bits(rng.normal(size=(96, 6, 64)).astype(np.float32), 30)[0])
    outs = [gpu.buffer(96 * 6 * 64 * 2) for _ in range(3)]
    for out in outs:
        gpu.kv8_attention(buffers, [s.context for s in states], lengths, rows, 6, 2, 64, 1, 0.125, q, out, 30)
    got = [gpu.read(out, np.int16, (96 * 6 * 64,)) for out in outs]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    for b in buffers + [q] + outs:
        gpu.release(b)
