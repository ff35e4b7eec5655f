"""8-bit K/V rows and masked attention at the ends of what they take, against the definition in 64 bits."""
import numpy as np
import pytest

from kv8_util import EPS, TOP, State, attention, evict, from_bits, random_state, rounded, state_bytes, to_bits
from test_gpu_kv8_attention import attend, check

pytestmark = pytest.mark.gpu


# ---- what lies behind the last row ----

def spoiled(rng, context, kv_heads, dim, code, length, fill):
    """A state whose rows behind `length` and whose blocks' scales behind it are as some other use left them (0x7f and 0xff are NaN in E4M3)."""
    state = State(context, kv_heads, dim, code, fill=fill)
    state.scales[:] = np.nan
    if length:
        x = rng.normal(size=(2, length, kv_heads, dim)).astype(np.float32)
        state.write(0, x[0], x[1])
    return state


@pytest.mark.parametrize("fill", [0x7f, 0xff])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (128, 8, 2), (256, 6, 2)])
@pytest.mark.parametrize("rows", [1, 4, 70])
def test_what_lies_behind_the_last_row_does_not_count(gpu, fill, code, dim, heads, kv_heads, rows):
    rng = np.random.default_rng(dim + rows + fill + code)
    lengths = [1, 15, 16, 17, 31, 32, 33, 700, 0, 2049]
    states = [spoiled(rng, rounded(n + 33), kv_heads, dim, code, n, fill) for n in lengths]
    for kind in (1, 30):
        check(gpu, states, lengths, [rows] * len(lengths), heads, kind, rng, weights=rows < 70)
    check(gpu, states, lengths, [rows] * len(lengths), heads, 1, rng, window=20, cap=9.0, prefixes=[n // 2 for n in lengths])


@pytest.mark.parametrize("fill", [0x7f, 0xff])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,keep", [(64, 45), (128, 33), (256, 50)])
def test_attention_over_an_eviction_into_memory_of_another_use(gpu, fill, code, dim, keep):
    rng = np.random.default_rng(dim + keep + fill)
    n, kv_heads, heads, context = 150, 2, 4, 96
    x = rng.normal(size=(2, n, kv_heads, dim)).astype(np.float32)
    state = State(160, kv_heads, dim, code).write(0, x[0], x[1])
    weights = rng.uniform(size=(kv_heads, 160)).astype(np.float32)
    source, w = gpu.upload(state.pack()), gpu.upload(weights)
    target, moved = gpu.upload(np.full(state_bytes(context, kv_heads, dim), fill, np.uint8)), gpu.buffer(kv_heads * context * 4)
    gpu.kv8_evict([source], [160], [n], [w], keep, 3, 9, kv_heads, dim, code, [target], [context], [moved])
    host, _, _ = evict(state, n, weights, keep, 3, 9)
    for rows in (1, 6, 40):
        raw, held = to_bits(rng.normal(size=(rows, heads, dim)).astype(np.float32), 30)
        q, out = gpu.upload(raw), gpu.buffer(rows * heads * dim * 2)
        gpu.kv8_attention([target], [context], [keep], [rows], heads, kv_heads, dim, code, dim ** -0.5, q, out, 30)
        got = from_bits(gpu.read(out, np.int16, (rows, heads, dim)), 30)
        want, _, size = attention(held, *host.values(keep), dim ** -0.5)
        assert np.all(np.abs(got - want) <= EPS[30] * np.abs(want) + (EPS[30] + 2.0 ** -16) * size + 1e-7), rows
        for b in (q, out):
            gpu.release(b)
    for b in (source, w, target, moved):
        gpu.release(b)


# ---- value scales far apart and far down ----

def bound(kind, held, state, length, want, size, heads, lowest=0.0, **rule):
    """What an output may be off, from what its own row sees: its rounding; the weights' (half a step of FP16 or BF16) and 2^-16 of the sum of |p v| for
    the FP32 arithmetic, as in kv8_util.tolerance; and, since a weight times its block's scale enters the products at 2^7 times its share of the row's largest
    or more, half of 2^-24 a key of that (codes of up to TOP): TOP * 2^-32 * n of the largest product, which is at most their sum. `lowest`: what a
    value scale may be off at the low end, TOP times it a value. Outputs below the normal numbers of F16: half of 2^-24."""
    k, _ = state.values(length)
    scales = np.repeat(state.scales[state.kv_heads:], 32, 1)[:, :length].T[:, :, None].astype(np.float64)
    products, _, _ = attention(held, k, np.broadcast_to(scales, (length, state.kv_heads, held.shape[2])), held.shape[2] ** -0.5, **rule)
    return (EPS[kind] * np.abs(want) + (EPS[kind] + 2.0 ** -16) * size + TOP[state.code] * 2.0 ** -32 * length * products + TOP[state.code] * lowest +
            (2.0 ** -25 if kind == 1 else 0.0))


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,rows", [(64, 300), (128, 290), (256, 70), (128, 7), (64, 1), (256, 2)])
@pytest.mark.parametrize("where", ["later", "left", "light"])
def test_a_block_of_large_values_that_a_row_gives_no_weight(gpu, kind, code, dim, rows, where):
    # one block 2^23 times the others, behind a row's position, left by its window, or at a distance that leaves it nothing
    rng = np.random.default_rng(dim + rows + code)
    n, heads, kv_heads = 512, 4, 2
    x = rng.normal(size=(2, n, kv_heads, dim)).astype(np.float32)
    x[1] *= 2.0 ** -9
    large = slice(480, 512) if where == "later" else slice(0, 32)
    x[1, large] *= 2.0 ** 23
    state = State(n, kv_heads, dim, code).write(0, x[0], x[1])
    rule = {"later": {}, "left": dict(window=100), "light": dict(slopes=np.full(heads, 0.6, np.float32))}[where]
    q = rng.normal(size=(rows, heads, dim)).astype(np.float32)
    got, _, held = attend(gpu, [state], [n], [rows], heads, q, kind, **rule)
    want, _, size = attention(held, *state.values(n), dim ** -0.5, **rule)
    limit = bound(kind, held, state, n, want, size, heads, **rule)
    assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())


# ---- key scales far down ----

@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 4), (256, 1), (64, 80), (128, 100), (256, 70)])
@pytest.mark.parametrize("size", [1e-20, 1e-31, 1e-34])
def test_small_keys_under_large_queries(gpu, dim, rows, size):
    rng = np.random.default_rng(dim + rows)
    n, heads, kv_heads = 300, 4, 2
    x = rng.normal(size=(2, n, kv_heads, dim)).astype(np.float32)
    x[0] *= np.float32(size)
    state = State(320, kv_heads, dim, 0).write(0, x[0], x[1])
    q = (rng.normal(size=(rows, heads, dim)) / size).astype(np.float32)
    for rule in (dict(), dict(cap=3.0), dict(slopes=np.full(heads, 0.01, np.float32), window=150)):
        got, _, held = attend(gpu, [state], [n], [rows], heads, q, 30, **rule)
        want, _, total = attention(held, *state.values(n), dim ** -0.5, **rule)
        limit = bound(30, held, state, n, want, total, heads, **rule)
        assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())


@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 4), (256, 1)])
def test_the_largest_queries(gpu, dim, rows):
    # BF16 rows of up to 2^127 over keys of 1e-36
    rng = np.random.default_rng(dim + rows)
    n, heads, kv_heads = 300, 4, 2
    x = rng.uniform(-1, 1, size=(2, n, kv_heads, dim)).astype(np.float32)
    x[0] *= np.float32(1e-36)
    state = State(320, kv_heads, dim, 0).write(0, x[0], x[1])
    q = (rng.uniform(-1, 1, size=(rows, heads, dim)) * 2.0 ** 119).astype(np.float32)
    q[0, 0] *= 2.0 ** -8
    q[0, 1, 3] = 1.7e38
    got, _, held = attend(gpu, [state], [n], [rows], heads, q, 30)
    want, _, total = attention(held, *state.values(n), dim ** -0.5)
    limit = bound(30, held, state, n, want, total, heads)
    assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())


# ---- small values ----

@pytest.mark.parametrize("magnitude", [1e30, 1.0, 1e-8, 1e-20, 1e-30, 1e-34])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 3), (256, 2), (64, 80), (128, 100), (256, 70)])
@pytest.mark.parametrize("zeros", [slice(0, 32), slice(96, 160), slice(0, 0)])
def test_small_and_large_values_beside_blocks_of_zeros(gpu, magnitude, dim, rows, zeros):
    # a block of zeros weighs like any other and takes nothing from the rest; head 1: a few blocks of ones beside the small or large ones
    rng = np.random.default_rng(dim + rows)
    n, heads, kv_heads, copies = 1000, 4, 2, 64 if rows < 10 else 1   # (copies: so many tiles that a warp has several)
    x = rng.normal(size=(2, n, kv_heads, dim)).astype(np.float32)
    x[1, :, 0] *= np.float32(magnitude)
    x[1, 32:96, 1] *= np.float32(magnitude)
    x[1, zeros] = 0
    state = State(1024, kv_heads, dim, 0).write(0, x[0], x[1])
    q = rng.normal(size=(copies * rows, heads, dim)).astype(np.float32)
    got, _, held = attend(gpu, [state] * copies, [n] * copies, [rows] * copies, heads, q, 30)
    for copy in range(0, copies, 21):
        at = slice(copy * rows, copy * rows + rows)
        want, _, size = attention(held[at], *state.values(n), dim ** -0.5)
        # (half of 2^-24 a key under 2^7 times 2^-88: what a product with a smaller scale may lose of itself)
        limit = bound(30, held[at], state, n, want, size, heads, lowest=n * 2.0 ** (-25 - 7 - 88))
        assert np.all(np.abs(got[at] - want) <= limit), (copy, float((np.abs(got[at] - want) / limit).max()))


# ---- arrays that overlap or lie askew ----

def test_nothing_written_lies_over_what_is_read(gpu):
    from straydog_b200.backend import StraydogError
    size = state_bytes(64, 1, 64)
    pool = gpu.upload(np.zeros(8 * size, np.uint8))
    one = dict(heads=1, kv_heads=1, dim=64, code=0, scale=0.1, type=1)
    q, out, slopes, weights = pool.at(2 * size), pool.at(3 * size), pool.at(4 * size), pool.at(5 * size)
    good = dict(states=[pool], contexts=[64], lengths=[9], rows=[1], q=q, out=out, slopes=slopes, weights=[weights], **one)
    two = dict(states=[pool, pool.at(size)], contexts=[64] * 2, lengths=[9] * 2, rows=[1] * 2, weights=[weights, pool.at(6 * size)])
    bad = [dict(weights=[pool.pointer]), dict(weights=[pool.at(2 * 64 * 64)]), dict(weights=[q]), dict(weights=[q + 124]), dict(weights=[slopes]), dict(slopes=out),
           dict(slopes=out + 124), dict(two, weights=[weights, pool.at(2 * size - 256)]), dict(two, weights=[pool.at(size), weights]), dict(two, out=weights)]
    for change in bad:
        with pytest.raises(StraydogError, match="overlap|lies over"):
            gpu.kv8_attention(**{**good, **change})
    with pytest.raises(StraydogError, match="overlap|lies over"):
        gpu.masked_attention(q, pool.pointer, pool.at(size), out, [1], [4], 1, 1, 64, 1, 0.1, slopes=out + 64)
    assert not np.any(gpu.read(pool, np.uint8, (8 * size,)))
    gpu.kv8_attention(**good)
    gpu.kv8_attention(**{**good, **two})
    gpu.kv8_attention(**{**good, "slopes": q})   # (what is read may be read twice)
    gpu.release(pool)


def test_slopes_lie_on_four_byte_boundaries(gpu):
    from straydog_b200.backend import StraydogError
    state, q, out, slopes = gpu.buffer(state_bytes(64, 1, 64)), gpu.buffer(128), gpu.upload(np.full(64, 0x5a5a, np.int16)), gpu.buffer(64)
    for off in (1, 2, 3, 6):
        with pytest.raises(StraydogError, match="slopes"):
            gpu.kv8_attention([state], [64], [9], [1], 1, 1, 64, 0, 0.1, q, out, 1, slopes=slopes.at(off))
        with pytest.raises(StraydogError, match="slopes"):
            gpu.masked_attention(q, state.pointer, state.pointer, out, [1], [4], 1, 1, 64, 1, 0.1, slopes=slopes.at(off))
    assert np.all(gpu.read(out, np.int16, (64,)) == 0x5a5a)
    for b in (state, q, out, slopes):
        gpu.release(b)


# ---- scores far past a cap ----

@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 3), (256, 1), (64, 90), (128, 80), (256, 70)])
@pytest.mark.parametrize("cap", [1e3, 1e5])
def test_a_score_far_under_a_large_cap_leaves_the_others_theirs(gpu, kind, dim, rows, cap):
    # keys with scores of -cap / 3: their weight is 0, and the others' scores, of a few units under the cap's curve, are as exact as without them
    rng = np.random.default_rng(dim + rows)
    n, heads, kv_heads = 256, 4, 2
    k, v = (rng.normal(size=(n, kv_heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(rows, heads, dim)).astype(np.float32)
    q[:, :, 0], k[:, :, 0] = 16.0, 0.0
    k[3::64] = 0.0
    k[3::64, :, 0] = -cap / 3 * dim ** 0.5 / 16
    v[3::64] = 0.0
    (qr, qh), (kr, kh), (vr, vh) = (to_bits(x, kind) for x in (q, k, v))
    buffers = [gpu.upload(x) for x in (qr, kr, vr)]
    out = gpu.buffer(rows * heads * dim * 2)
    gpu.masked_attention(*(b.pointer for b in buffers), out, [rows], [n], heads, kv_heads, dim, kind, dim ** -0.5, cap=cap)
    got = from_bits(gpu.read(out, np.int16, (rows, heads, dim)), kind)
    want, _, size = attention(qh, kh, vh, dim ** -0.5, cap=cap)
    limit = EPS[kind] * np.abs(want) + (EPS[kind] + 2.0 ** -16) * size + 1e-7
    assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())
    for b in buffers + [out]:
        gpu.release(b)
    # 8-bit rows: the same over the codes that the small keys keep (blocks of their own for the large ones)
    k[:32], k[32:] = np.concatenate([k[3::64]] * 8), np.where(np.arange(224)[:, None, None] % 64 == 35, 0, k[32:])
    state = State(n, kv_heads, dim, 0).write(0, k, v)
    got, _, held = attend(gpu, [state], [n], [rows], heads, q, kind, cap=cap)
    want, _, size = attention(held, *state.values(n), dim ** -0.5, cap=cap)
    limit = EPS[kind] * np.abs(want) + (EPS[kind] + 2.0 ** -16) * size + 1e-7
    assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())


# ---- the bits of a chunk's weights ----

@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(64, 6, 2, 70), (128, 8, 2, 150), (256, 4, 1, 90), (128, 8, 1, 8), (64, 4, 4, 1)])
def test_weights_under_bf16_rows_keep_eleven_bits(gpu, code, dim, heads, kv_heads, rows):
    # few rows and chunks alike: all but the output's own rounding is FP16's (half a step of each weight, 2^-16 for the FP32 arithmetic, small products)
    rng = np.random.default_rng(dim + rows + code)
    lengths, chunk = [700, 300, 64], [rows, max(rows // 2, 1), rows]
    states = [random_state(rng, rounded(n), kv_heads, dim, code, n) for n in lengths]
    for size in (1.0, 1e-20):   # (rows of any size: a power of two brings them to FP16)
        q = (rng.normal(size=(sum(chunk), heads, dim)) * size).astype(np.float32)
        got, _, held = attend(gpu, states, lengths, chunk, heads, q, 30)
        row = 0
        for state, n, r in zip(states, lengths, chunk):
            at = slice(row, row + r)
            want, _, total = attention(held[at], *state.values(n), dim ** -0.5)
            limit = bound(1, held[at], state, n, want, total, heads) + EPS[30] * np.abs(want)
            assert np.all(np.abs(got[at] - want) <= limit), (size, n, float((np.abs(got[at] - want) / limit).max()))
            row += r


@pytest.mark.parametrize("dim,rows", [(64, 80), (128, 100), (256, 70)])
def test_the_largest_queries_of_a_chunk(gpu, dim, rows):
    # BF16 rows of up to 2^127 over keys of 1e-36, some rows small or zero
    rng = np.random.default_rng(dim + rows)
    n, heads, kv_heads = 300, 4, 2
    x = rng.uniform(-1, 1, size=(2, n, kv_heads, dim)).astype(np.float32)
    x[0] *= np.float32(1e-36)
    state = State(320, kv_heads, dim, 0).write(0, x[0], x[1])
    q = (rng.uniform(-1, 1, size=(rows, heads, dim)) * 2.0 ** 119).astype(np.float32)
    q[0, 0] *= 2.0 ** -8
    q[0, 1, 3] = 1.7e38
    q[5], q[6] = 0.0, 1e-39
    for rule in (dict(), dict(cap=3.0), dict(slopes=np.full(heads, 0.01, np.float32), window=150)):
        got, _, held = attend(gpu, [state], [n], [rows], heads, q, 30, **rule)
        want, _, total = attention(held, *state.values(n), dim ** -0.5, **rule)
        limit = bound(30, held, state, n, want, total, heads, **rule)
        assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())


def test_chunks_of_bf16_rows_between_others(gpu):
    # what is lifted begins with the first chunk's rows and has the others' between; more chunks than a launch takes
    rng = np.random.default_rng(8)
    lengths, rows = [90, 200, 40, 0, 300, 60] * 20, [2, 50, 3, 40, 64, 0] * 20
    some = [random_state(rng, 320, 2, 128, 1, n) for n in lengths[:6]]
    check(gpu, some * 20, lengths, rows, 6, 30, rng, q_pad=16, out_pad=8)


@pytest.mark.parametrize("scale,cap", [(1e20, 1e-20), (0.1, 1e-40), (1e29, 0.01)])
def test_a_cap_far_below_the_scale_is_refused(gpu, scale, cap):
    # scale / cap past 1e30: a score of 0 would be a NaN
    from straydog_b200.backend import StraydogError
    state, q, out = gpu.buffer(state_bytes(64, 1, 64)), gpu.buffer(128), gpu.upload(np.full(64, 0x5a5a, np.int16))
    with pytest.raises(StraydogError, match="cap"):
        gpu.kv8_attention([state], [64], [9], [1], 1, 1, 64, 0, scale, q, out, 1, cap=cap)
    with pytest.raises(StraydogError, match="cap"):
        gpu.masked_attention(q, state.pointer, state.pointer, out, [1], [4], 1, 1, 64, 1, scale, cap=cap)
    assert np.all(gpu.read(out, np.int16, (64,)) == 0x5a5a)
    for b in (state, q, out):
        gpu.release(b)


def test_memory_that_cannot_be_had_is_that_calls_error_alone(gpu):
    # places for 8 x 1024 x 2^24 kept positions are 550 GB: refused. The calls behind it go on, and what they report is their own.
    from straydog_b200.backend import StraydogError
    rng = np.random.default_rng(3)
    count, kv_heads, dim = 8, 1024, 64
    states, targets = ([gpu.buffer(state_bytes(32, kv_heads, dim)) for _ in range(count)] for _ in range(2))
    weights, moved = ([gpu.buffer(kv_heads * 32 * 4) for _ in range(count)] for _ in range(2))
    with pytest.raises(StraydogError, match="memory"):
        gpu.kv8_evict(states, [32] * count, [9] * count, weights, 1 << 24, 0, 0, kv_heads, dim, 0, targets, [32] * count, moved)
    gpu.kv8_evict(states, [32] * count, [9] * count, weights, 8, 0, 0, kv_heads, dim, 0, targets, [32] * count, moved)
    small = random_state(rng, 96, 2, dim, 1, 70)
    check(gpu, [small], [70], [3], 4, 1, rng, weights=True)
    for b in states + targets + weights + moved:
        gpu.release(b)
