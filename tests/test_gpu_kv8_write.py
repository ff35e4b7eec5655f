"""sdx_kv8_write (8-bit K/V rows with one scale a block of 32 positions and head) against the definition, bit for bit."""
import numpy as np
import pytest

from kv8_util import State, random_state, rounded, state_bytes, to_bits

pytestmark = pytest.mark.gpu


def upload_state(gpu, state, guard=64):
    raw = state.pack()
    return gpu.upload(np.concatenate([raw, np.full(guard, 0xA5, np.uint8)]))


def download_state(gpu, buffer, state, guard=64):
    raw = gpu.read(buffer, np.uint8, (state.pack().size + guard,))
    assert np.all(raw[-guard:] == 0xA5), "guard behind the state"
    return state.unpack(raw[:-guard])


def assert_same(got, want):
    assert np.array_equal(got.scales.view(np.uint32), want.scales.view(np.uint32))
    if want.code == 1:   # (the two zeros of E4M3 are one value)
        assert np.array_equal(np.where(got.codes == 0x80, 0, got.codes), np.where(want.codes == 0x80, 0, want.codes))
    else:
        assert np.array_equal(got.codes, want.codes)


def rows_of(rng, steps, kv_heads, dim, kind, spread=2.0):
    x = rng.normal(size=(steps, kv_heads, dim)) * np.exp2(spread * rng.normal(size=(steps, 1, 1)))
    raw, held = to_bits(x.astype(np.float32), kind)
    return raw, held.astype(np.float32)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("kind", [0, 1, 30])
def test_appends_give_the_definitions_bits(gpu, dim, code, kind):
    # a prompt, single tokens into a begun block, a run over several borders, one that starts on a border: the states after all of them
    rng = np.random.default_rng(dim * 10 + code * 3 + kind)
    kv_heads, contexts = 3, [96, 160, 32]
    plans = [[(0, 33), (33, 1), (34, 30), (64, 32)], [(0, 1), (1, 1), (2, 100), (102, 58)], [(0, 5), (5, 1), (6, 1), (7, 25)]]
    want = [State(c, kv_heads, dim, code, fill=0x55) for c in contexts]
    states = [upload_state(gpu, s) for s in want]
    for step in range(4):
        bases, steps = [p[step][0] for p in plans], [p[step][1] for p in plans]
        keys, values = (rows_of(rng, sum(steps), kv_heads, dim, kind) for _ in range(2))
        k, v = gpu.upload(keys[0]), gpu.upload(values[0])
        gpu.kv8_write(states, contexts, bases, steps, kv_heads, dim, code, k, v, kind)
        row = 0
        for s in range(3):
            want[s].write(bases[s], keys[1][row:row + steps[s]], values[1][row:row + steps[s]])
            row += steps[s]
            assert_same(download_state(gpu, states[s], want[s]), want[s])
        for b in (k, v):
            gpu.release(b)
    for b in states:
        gpu.release(b)


def test_rows_of_a_wider_projection_and_sequences_without_rows(gpu):
    rng = np.random.default_rng(3)
    kv_heads, dim, code, kind, n = 2, 128, 0, 30, 70   # (more sequences than one launch takes)
    steps = [0 if s % 5 == 2 else 1 + s % 3 for s in range(n)]
    bases = [(7 * s) % 29 for s in range(n)]
    want = [random_state(rng, 64, kv_heads, dim, code, bases[s]) for s in range(n)]
    states = [upload_state(gpu, s) for s in want]
    fused, held = rows_of(rng, sum(steps), 2 * kv_heads + 1, dim, kind)   # [key heads | value heads | one more]
    buffer = gpu.upload(fused)
    gpu.kv8_write(states, [64] * n, bases, steps, kv_heads, dim, code, buffer.at(0), buffer.at(kv_heads * dim * 2), kind, stride=(2 * kv_heads + 1) * dim)
    row = 0
    for s in range(n):
        if steps[s]:
            want[s].write(bases[s], held[row:row + steps[s], :kv_heads], held[row:row + steps[s], kv_heads:2 * kv_heads])
        row += steps[s]
        assert_same(download_state(gpu, states[s], want[s]), want[s])
    for b in states + [buffer]:
        gpu.release(b)


@pytest.mark.parametrize("code", [0, 1])
def test_zeros_infinities_nan_and_tiny_values(gpu, code):
    x = np.zeros((40, 1, 64), np.float32)
    x[1, 0, :4] = [np.inf, -np.inf, np.nan, 3.0]
    x[33, 0, :6] = [1e-44, -1e-45, 0.0, -0.0, 1e-40, 2e-38]
    y = np.full((40, 1, 64), 3e38, np.float32)
    y[5] = np.nan
    want = State(64, 1, 64, code)
    state = upload_state(gpu, want)
    k, v = gpu.upload(x), gpu.upload(y)
    gpu.kv8_write([state], [64], [0], [40], 1, 64, code, k, v, 0)
    want.write(0, x, y)
    got = download_state(gpu, state, want)
    assert_same(got, want)
    assert not np.any((got.codes & 0x7f) == 0x7f) or code == 0   # (no NaN code)
    for b in (state, k, v):
        gpu.release(b)


def test_the_same_rows_again_change_nothing(gpu):
    rng = np.random.default_rng(8)
    want = random_state(rng, 64, 2, 64, 0, 20)
    state = upload_state(gpu, want)
    raw, held = rows_of(rng, 9, 2, 64, 0)
    buffer = gpu.upload(raw)
    gpu.kv8_write([state], [64], [20], [9], 2, 64, 0, buffer, buffer, 0)
    first = download_state(gpu, state, want)
    gpu.kv8_write([state], [64], [20], [9], 2, 64, 0, buffer, buffer, 0)
    assert_same(download_state(gpu, state, want), first)
    assert_same(first, want.write(20, held, held))
    for b in (state, buffer):
        gpu.release(b)


def test_refusals_leave_the_states_alone(gpu):
    from straydog_b200.backend import StraydogError
    size = state_bytes(64, 2, 128)
    state = gpu.upload(np.full(size, 0x33, np.uint8))
    other = gpu.buffer(size)
    rows = gpu.buffer(64 * 2 * 128 * 4)
    good = dict(states=[state], contexts=[64], bases=[0], steps=[4], kv_heads=2, dim=128, code=0, keys=rows.pointer, values=rows.pointer, type=0, stride=0)
    bad = [dict(contexts=[48]), dict(contexts=[0]), dict(contexts=[128]), dict(bases=[61]), dict(bases=[65], steps=[0]), dict(bases=[2 ** 63], steps=[2 ** 63]),
           dict(dim=96), dict(kv_heads=0), dict(code=2), dict(type=2), dict(stride=255), dict(stride=257), dict(keys=rows.pointer + 4),
           dict(states=[state.pointer + 8]), dict(states=[state, state], contexts=[64] * 2, bases=[0] * 2, steps=[4] * 2), dict(keys=None),
           dict(values=state.pointer), dict(steps=[65]), dict(keys=rows.at(62 * 1024)), dict(states=[], contexts=[], bases=[], steps=[])]
    for change in bad:
        with pytest.raises(StraydogError):
            gpu.kv8_write(**{**good, **change})
    assert np.all(gpu.read(state, np.uint8, (size,)) == 0x33)
    gpu.kv8_write(**{**good, "steps": [0]})   # (nothing to write is no error)
    assert np.all(gpu.read(state, np.uint8, (size,)) == 0x33)
    for b in (state, other, rows):
        gpu.release(b)


def test_size_of_a_state(gpu):
    assert gpu.kv8_bytes(64, 2, 128) == state_bytes(64, 2, 128) and rounded(33) == 64
