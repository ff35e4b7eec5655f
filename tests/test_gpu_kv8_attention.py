"""sdx_kv8_attention (decode, verification rows and prompt chunks over 8-bit K/V rows with block scales) against the definition in 64 bits."""
import numpy as np
import pytest

from kv8_util import State, attention, from_bits, random_state, rounded, state_bytes, to_bits, tolerance

pytestmark = pytest.mark.gpu
GUARD = 64


def attend(gpu, states, lengths, rows, heads, q, kind, weights=None, q_pad=0, out_pad=0, **rule):
    """states: host States; q: [total][heads][dim] float32. Returns (out as float64, weights)."""
    dim, kv_heads, code = states[0].dim, states[0].kv_heads, states[0].code
    total, width = q.shape[0], heads * dim
    raw, held = to_bits(q, kind)
    padded = np.full((total, width + q_pad), 0x7fff, np.int16)   # (a NaN beside the rows)
    padded[:, :width] = raw.reshape(total, width)
    buffers = [gpu.upload(s.pack()) for s in states]
    q_buffer = gpu.upload(padded)
    out = gpu.upload(np.full(total * (width + out_pad) + GUARD, 0x5a5a, np.int16))
    slopes = rule.pop("slopes", None)
    slope_buffer = gpu.upload(np.asarray(slopes, np.float32)) if slopes is not None else None
    weight_buffers = [gpu.upload(w) for w in weights] if weights else None
    gpu.kv8_attention(buffers, [s.context for s in states], lengths, rows, heads, kv_heads, dim, code, dim ** -0.5, q_buffer, out, kind,
                      slopes=slope_buffer, weights=weight_buffers, q_stride=width + q_pad, out_stride=width + out_pad, **rule)
    got = gpu.read(out, np.int16, (total * (width + out_pad) + GUARD,))
    assert gpu.decode_status() == 0
    got, guard = got[:-GUARD].reshape(total, width + out_pad), got[-GUARD:]
    assert np.all(guard == 0x5a5a) and np.all(got[:, width:] == 0x5a5a), "what lies beside the output"
    summed = [gpu.read(b, np.float32, w.shape) for b, w in zip(weight_buffers, weights)] if weights else None
    for b in buffers + [q_buffer, out, slope_buffer] + (weight_buffers or []):
        if b:
            gpu.release(b)
    return from_bits(np.ascontiguousarray(got[:, :width]), kind).reshape(total, heads, dim), summed, held


def check(gpu, states, lengths, rows, heads, kind, rng, prefixes=None, weights=False, **rule):
    dim = states[0].dim
    q = rng.normal(size=(sum(rows), heads, dim)).astype(np.float32)
    before = [rng.uniform(0, 2, size=(s.kv_heads, s.context)).astype(np.float32) for s in states] if weights else None
    extra = {"prefixes": prefixes} if prefixes else {}
    pads = dict(q_pad=rule.pop("q_pad", 0), out_pad=rule.pop("out_pad", 0))
    got, summed, held = attend(gpu, states, lengths, rows, heads, q, kind, before, **pads, **extra, **rule)
    row = 0
    for s, (state, length, r) in enumerate(zip(states, lengths, rows)):
        k, v = state.values(length)
        want, sums, size = attention(held[row:row + r], k, v, dim ** -0.5, prefix=prefixes[s] if prefixes else 0, **rule)
        off = np.abs(got[row:row + r] - want)
        assert np.all(off <= tolerance(kind, want, size)), (s, length, r, float((off / tolerance(kind, want, size)).max()))
        if weights and r:
            full = np.zeros_like(before[s], np.float64)
            full[:, :length] = sums
            # (exponentials and scores as in `tolerance`, relative to each weight, and the sum's own rounding)
            assert np.all(np.abs(summed[s] - (before[s] + full)) <= 2.0 ** -16 * full + 2.0 ** -23 * (before[s] + full)), s
            assert np.array_equal(summed[s][:, length:], before[s][:, length:])
        row += r


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (64, 48, 3), (128, 8, 1), (128, 32, 2), (256, 16, 2), (256, 24, 2)])
def test_one_token_of_ragged_sequences(gpu, kind, code, dim, heads, kv_heads):
    rng = np.random.default_rng(dim + heads + code + kind)
    lengths = [1, 31, 0, 33, 700, 32, 2049]
    states = [random_state(rng, rounded(max(n, 1)), kv_heads, dim, code, n) for n in lengths]
    check(gpu, states, lengths, [1] * len(lengths), heads, kind, rng)


@pytest.mark.parametrize("rule", [dict(cap=3.0), dict(slopes=True), dict(window=1), dict(window=40), dict(window=5000), dict(prefixes=[600, 3, 64, 0]),
                                  dict(window=33, prefixes=[70, 1, 100, 150]), dict(cap=5.0, slopes=True, window=100, prefixes=[1, 2, 3, 4])],
                         ids=lambda r: "-".join(r))
@pytest.mark.parametrize("dim,heads,kv_heads,most", [(64, 6, 2, 5), (128, 8, 2, 4), (256, 16, 2, 4), (128, 8, 2, 40), (256, 6, 2, 70), (64, 4, 1, 300)])
def test_rules_for_verification_rows_and_chunks(gpu, rule, dim, heads, kv_heads, most):
    rng = np.random.default_rng(dim + most + len(rule))
    rule = dict(rule)
    if rule.pop("slopes", None):
        rule["slopes"] = np.exp2(-np.arange(1, heads + 1) / 2).astype(np.float32)
    lengths, rows = [700, 5, 333, 160], [most, 1, max(1, most // 2), most]   # (the second: fewer keys than the chunk's first rows need)
    rows[1] = min(most, 9)
    states = [random_state(rng, rounded(n), kv_heads, dim, 0, n) for n in lengths]
    check(gpu, states, lengths, rows, heads, 30 if dim == 128 else 1, rng, q_pad=8 * 3, out_pad=8, **rule)


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(64, 5, 5, 129), (128, 12, 1, 65), (256, 8, 2, 131), (128, 128, 1, 3)])
def test_chunks(gpu, code, kind, dim, heads, kv_heads, rows):
    rng = np.random.default_rng(dim + rows)
    lengths = [rows, 1000, rows + 1, 0]
    states = [random_state(rng, rounded(max(n, 1)), kv_heads, dim, code, n) for n in lengths]
    check(gpu, states, lengths, [rows, rows, rows, rows], heads, kind, rng)


def test_a_batch_of_decode_rows_and_chunks_and_sequences_without_rows(gpu):
    rng = np.random.default_rng(5)
    lengths = [100, 300, 50, 290, 128] * 15   # (more sequences than a launch takes)
    rows = [1, 100, 0, 2, 128] * 15
    states = [random_state(rng, 320, 2, 64, 0, n) for n in lengths[:5]] * 15
    check(gpu, states, lengths, rows, 4, 1, rng)


@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(64, 8, 2, 1), (128, 8, 2, 4), (256, 16, 2, 1), (256, 16, 2, 2), (128, 8, 1, 8)])
@pytest.mark.parametrize("rule", [dict(), dict(window=50, prefixes=[40, 0, 3]), dict(cap=4.0, slopes=True)], ids=["plain", "window", "cap"])
def test_weights_are_added_up(gpu, dim, heads, kv_heads, rows, rule):
    rng = np.random.default_rng(dim + rows)
    rule = dict(rule)
    if rule.pop("slopes", None):
        rule["slopes"] = np.exp2(-np.arange(1, heads + 1) / 2).astype(np.float32)
    lengths = [333, 1, 2000]
    states = [random_state(rng, rounded(n) + 32, kv_heads, dim, 0, n) for n in lengths]
    check(gpu, states, lengths, [rows, 1, rows], heads, 30, rng, weights=True, **rule)


@pytest.mark.parametrize("dim,most", [(128, 1), (128, 64)])
def test_a_nan_query_row_stays_its_own(gpu, dim, most):
    rng = np.random.default_rng(1)
    state = random_state(rng, 256, 1, dim, 0, 200)
    q = rng.normal(size=(most + 1, 4, dim)).astype(np.float32)
    q[0, 1, 7] = np.nan
    for kind in (1, 30):
        got, _, held = attend(gpu, [state, state], [200, 150], [most, 1], 4, q, kind)
        want, _, size = attention(np.nan_to_num(held[:most]), *state.values(200), dim ** -0.5)
        assert np.all(np.isnan(got[0, 1]))
        off = np.abs(got[:most] - want) <= tolerance(kind, want, size)
        off[0, 1] = True
        assert np.all(off)


def test_large_and_small_queries(gpu):
    # BF16 rows that FP16 could not hold: the scores are exact all the same
    rng = np.random.default_rng(2)
    state = random_state(rng, 96, 1, 64, 0, 96, spread=0.0)
    q = rng.normal(size=(3, 2, 64)).astype(np.float32)
    for factor in (1e-30, 1e6):
        got, _, held = attend(gpu, [state], [96], [3], 2, q * np.float32(factor), 30)
        want, _, size = attention(held, *state.values(96), 64 ** -0.5)
        # (scores of 1e6 are off by 2^-22 of themselves: the winner's weight is 1 and the others' 0 either way unless two are within that)
        assert np.all(np.abs(got - want) <= tolerance(30, want, size) + (0.5 * size if factor > 1 else 0))


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 3), (256, 1), (64, 200), (128, 90), (256, 150)])
def test_blocks_whose_scales_are_far_apart(gpu, kind, dim, rows):
    # values of 2^-8 .. 2^8 from block to block, some blocks zero: the values' scales ride on the weights' exponents
    rng = np.random.default_rng(dim + rows)
    n = 400
    x = rng.normal(size=(2, n, 2, dim)).astype(np.float32)
    x[1] *= np.exp2(rng.integers(-8, 9, size=(13, 2, 1))).astype(np.float32).repeat(32, 0)[:n]
    x[:, 64:128] = 0
    state = State(416, 2, dim, 0).write(0, x[0], x[1])
    q = rng.normal(size=(rows, 4, dim)).astype(np.float32)
    got, _, held = attend(gpu, [state], [n], [rows], 4, q, kind)
    want, _, size = attention(held, *state.values(n), dim ** -0.5)
    # (a weight times its block's scale, over the largest such product, may lie below what FP16 holds as a normal number: half of 2^-24 a key)
    floor = 2.0 ** -25 * n * np.abs(state.values(n)[1]).max() if kind == 1 else 0.0
    assert np.all(np.abs(got - want) <= tolerance(kind, want, size) + floor)


@pytest.mark.parametrize("magnitude", [1e-37, 1e-20, 1e30])
@pytest.mark.parametrize("dim,rows", [(128, 1), (64, 3), (256, 2), (128, 100), (256, 70)])
def test_values_near_the_ends_of_fp32(gpu, dim, rows, magnitude):
    # scales down to subnormal ones, all of a head's or one block's: the sums of weights must not notice
    rng = np.random.default_rng(dim + rows)
    n = 200
    x = rng.normal(size=(2, n, 2, dim)).astype(np.float32)
    x[1, 64:96, 0] *= np.float32(magnitude)
    x[1, :, 1] *= np.float32(magnitude)
    state = State(224, 2, dim, 0).write(0, x[0], x[1])
    q = rng.normal(size=(rows, 4, dim)).astype(np.float32)
    got, _, held = attend(gpu, [state], [n], [rows], 4, q, 30)
    want, _, size = attention(held, *state.values(n), dim ** -0.5)
    # (without the absolute part of the tolerance, but scales below 2^-96, or 2^-64 of the head's largest, count as that: 127 times it a value)
    top = np.abs(x[1]).max(axis=(0, 2)).repeat(2)[None, :, None]
    assert np.all(np.abs(got - want) <= tolerance(30, want, size) - 1e-7 + 127 * 2.0 ** -96 + 2.0 ** -64 * top)


def test_zero_states(gpu):
    for rows in (1, 100):
        got, _, _ = attend(gpu, [State(128, 1, 64, 0)], [100], [rows], 1, np.ones((rows, 1, 64), np.float32), 1)
        assert np.all(got == 0)


def test_the_largest_head_layouts_and_a_long_sequence(gpu):
    rng = np.random.default_rng(11)
    n = 40000
    state = random_state(rng, rounded(n), 1, 64, 0, n, spread=0.0)
    check(gpu, [state], [n], [1], 8, 1, rng)
    check(gpu, [state], [n], [17], 4, 30, rng, window=30000)


def test_refusals(gpu):
    from straydog_b200.backend import StraydogError
    size = state_bytes(64, 2, 128)
    state, q = gpu.buffer(size), gpu.buffer(4 * 8 * 128 * 2)
    out = gpu.upload(np.full(4 * 8 * 128, 0x5a5a, np.int16))
    w = gpu.buffer(2 * 64 * 4)
    good = dict(states=[state], contexts=[64], lengths=[40], rows=[4], heads=8, kv_heads=2, dim=128, code=0, scale=0.1, q=q.pointer, out=out.pointer, type=1)
    bad = [dict(contexts=[63]), dict(lengths=[65]), dict(heads=7), dict(heads=0), dict(kv_heads=3), dict(dim=96), dict(code=-1), dict(type=0), dict(scale=0.0),
           dict(scale=float("nan")), dict(cap=-1.0), dict(cap=float("inf")), dict(q_stride=1016), dict(q_stride=1028), dict(out_stride=8), dict(q=q.pointer + 2),
           dict(out=out.pointer + 8), dict(rows=[5]), dict(q=out.pointer), dict(slopes=1), dict(weights=[w.pointer + 2]), dict(weights=[1]), dict(states=[0]),
           dict(states=[state] * 2, contexts=[64] * 2, lengths=[40] * 2, rows=[2] * 2, weights=[w] * 2), dict(rows=[2 ** 40]), dict(heads=512, kv_heads=2),
           dict(prefixes=[1, 2]), dict(rows=[4, 4])]
    for change in bad:
        with pytest.raises(StraydogError):
            gpu.kv8_attention(**{**good, **change})
    assert np.all(gpu.read(out, np.int16, (4 * 8 * 128,)) == 0x5a5a)
    big = gpu.buffer(17 * 8 * 128 * 2 * 2)
    with pytest.raises(StraydogError, match="64 query rows"):
        gpu.kv8_attention(**{**good, "rows": [17], "q": big.pointer, "out": big.at(17 * 8 * 128 * 2), "weights": [w]})
    gpu.kv8_attention(**{**good, "rows": [0]})
    assert np.all(gpu.read(out, np.int16, (4 * 8 * 128,)) == 0x5a5a)
    for b in (state, q, out, w, big):
        gpu.release(b)


def test_what_is_written_lies_apart(gpu):
    from straydog_b200.backend import StraydogError
    size = state_bytes(64, 1, 64)
    pool = gpu.upload(np.zeros(4 * size, np.uint8))
    q = gpu.buffer(2 * 64 * 2)
    one = dict(lengths=[9], rows=[1], heads=1, kv_heads=1, dim=64, code=0, scale=0.1, q=q.pointer, type=1)
    with pytest.raises(StraydogError, match="over a state"):
        gpu.kv8_attention([pool], [64], out=pool.at(size - 128), **one)
    with pytest.raises(StraydogError, match="over attention weights|over a state or"):
        gpu.kv8_attention([pool], [64], out=pool.at(2 * size), weights=[pool.at(2 * size + 64)], **one)
    with pytest.raises(StraydogError, match="overlap"):
        gpu.kv8_attention([pool] * 2, [64] * 2, [9] * 2, [1] * 2, 1, 1, 64, 0, 0.1, q.pointer, pool.at(3 * size), 1, weights=[pool.at(size), pool.at(size + 128)])
    with pytest.raises(StraydogError, match="overlap"):
        gpu.kv8_write([pool, pool.at(size - 16)], [64] * 2, [0] * 2, [1] * 2, 1, 64, 0, q.pointer, q.pointer, 1)
    assert not np.any(gpu.read(pool, np.uint8, (4 * size,)))
    gpu.kv8_attention([pool], [64], out=pool.at(size), weights=[pool.at(2 * size)], **one)   # (side by side is apart)
    for b in (pool, q):
        gpu.release(b)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (128, 8, 2), (256, 4, 1)])
@pytest.mark.parametrize("rows", [1, 5])
def test_one_long_sequence(gpu, dim, heads, kv_heads, rows):
    # a few rows over many partial sums, and an empty sequence beside it
    rng = np.random.default_rng(dim + rows)
    n = 9000
    states = [random_state(rng, rounded(n), kv_heads, dim, 0, n), random_state(rng, 32, kv_heads, dim, 0, 0)]
    check(gpu, states, [n, 0], [rows, 2], heads, 30, rng, weights=True)
    check(gpu, states, [n, 0], [rows, 2], heads, 1, rng, window=5000, cap=20.0)
