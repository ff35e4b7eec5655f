"""sdx_kv8_evict (the rows of greatest accumulated attention weight kept, moved together and rounded again where their new block's scale is larger)
against the definition, bit for bit."""
import numpy as np
import pytest

from kv8_util import State, evict, random_state, rounded, state_bytes

pytestmark = pytest.mark.gpu


def weights_of(rng, kv_heads, context, ties=0.3):
    w = np.exp(3 * rng.normal(size=(kv_heads, context))).astype(np.float32)
    return np.where(rng.uniform(size=w.shape) < ties, np.float32(0), w)


def check(gpu, states, lengths, weights, keep, sinks, recent, want_kept=True):
    n, kv_heads, dim, code = len(states), states[0].kv_heads, states[0].dim, states[0].code
    room = rounded(keep) + 32
    target = State(room, kv_heads, dim, code, fill=0x11)
    target.scales[:] = 7.0
    buffers = [gpu.upload(s.pack()) for s in states]
    w = [gpu.upload(x) for x in weights]
    targets = [gpu.upload(target.pack()) for _ in states]
    tw = [gpu.upload(np.full((kv_heads, room), -5, np.float32)) for _ in states]
    kept = gpu.upload(np.full((n, kv_heads, keep), -9, np.int32))
    gpu.kv8_evict(buffers, [s.context for s in states], lengths, w, keep, sinks, recent, kv_heads, dim, code, targets, [room] * n, tw,
                  kept if want_kept else None)
    positions = gpu.read(kept, np.int32, (n, kv_heads, keep))
    for s, (state, length) in enumerate(zip(states, lengths)):
        want, at, moved = evict(state, length, weights[s], keep, sinks, recent)
        count = at.shape[1]
        if want_kept:
            assert np.array_equal(positions[s, :, :count], at), s
            assert np.all(positions[s, :, count:] == -9)
        else:
            assert np.all(positions == -9)
        got_w = gpu.read(tw[s], np.float32, (kv_heads, room))
        assert np.array_equal(got_w[:, :count].view(np.uint32), moved.view(np.uint32)) and np.all(got_w[:, count:] == -5)
        got = target.unpack(gpu.read(targets[s], np.uint8, (target.pack().size,)))
        blocks = -(-count // 32)
        assert np.array_equal(got.scales[:, :blocks], want.scales[:, :blocks]) and np.all(got.scales[:, blocks:] == 7)
        a, b = got.codes[:, :count], want.codes[:, :count]
        if code == 1:
            a, b = np.where(a == 0x80, 0, a), np.where(b == 0x80, 0, b)
        assert np.array_equal(a, b) and np.all(got.codes[:, count:] == 0x11)
        assert np.array_equal(gpu.read(buffers[s], np.uint8, (state.pack().size,)), state.pack())
    for b in buffers + w + targets + tw + [kept]:
        gpu.release(b)


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("dim,kv_heads", [(64, 1), (128, 3), (256, 2)])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (33, 0, 33), (64, 4, 16), (100, 50, 50), (301, 4, 100), (2048, 1, 2)])
def test_ragged_sequences(gpu, code, dim, kv_heads, keep, sinks, recent):
    rng = np.random.default_rng(dim + keep)
    lengths = [keep + 1, 1, keep, 3 * keep + 7, 0, 2500]
    states = [random_state(rng, rounded(max(n, 1)), kv_heads, dim, code, n) for n in lengths]
    check(gpu, states, lengths, [weights_of(rng, kv_heads, s.context) for s in states], keep, sinks, recent)


@pytest.mark.parametrize("length", [1100, 5000, 40000, 300000])
def test_long_sequences(gpu, length):
    # (one block a head, a cluster of blocks, weights held in registers and read again)
    rng = np.random.default_rng(length)
    state = random_state(rng, rounded(length), 1, 64, 0, length, spread=0.5)
    check(gpu, [state], [length], [weights_of(rng, 1, state.context, ties=0.6)], length // 2, 4, 128)


@pytest.mark.parametrize("values", [[0.0], [0.0, -0.0, 1.0], [np.nan, 0.0, 1.0], [np.inf, -np.inf, np.nan, 2.0, -3.0], [np.nan]])
def test_ties_nan_and_infinities(gpu, values):
    rng = np.random.default_rng(6)
    lengths = [500, 3000]
    states = [random_state(rng, rounded(n), 2, 64, 0, n) for n in lengths]
    weights = [rng.choice(np.asarray(values, np.float32), size=(2, s.context)) for s in states]
    check(gpu, states, lengths, weights, 200, 3, 40)
    check(gpu, states, lengths, weights, 200, 3, 40, want_kept=False)


def test_more_sequences_than_a_launch_takes(gpu):
    rng = np.random.default_rng(7)
    state = random_state(rng, 128, 2, 64, 0, 128)
    lengths = [20 + s for s in range(70)]
    check(gpu, [state] * 70, lengths, [weights_of(rng, 2, 128) for _ in range(70)], 40, 2, 8)


def test_refusals_write_nothing(gpu):
    from straydog_b200.backend import StraydogError
    state, target = gpu.buffer(state_bytes(64, 2, 64)), gpu.upload(np.full(state_bytes(32, 2, 64), 0x22, np.uint8))
    w, tw, kept = gpu.buffer(2 * 64 * 4), gpu.buffer(2 * 32 * 4), gpu.buffer(2 * 32 * 4)
    good = dict(states=[state], contexts=[64], lengths=[64], weights=[w], keep=32, sinks=1, recent=4, kv_heads=2, dim=64, code=0, targets=[target],
                target_contexts=[32], target_weights=[tw], kept=kept)
    bad = [dict(contexts=[65]), dict(lengths=[65]), dict(keep=0), dict(keep=33), dict(sinks=33), dict(sinks=30, recent=3), dict(recent=2 ** 40), dict(dim=65), dict(code=3),
           dict(targets=[state]), dict(targets=[None]), dict(target_contexts=[64]), dict(target_contexts=[16]), dict(target_weights=[w]), dict(target_weights=[tw.pointer + 1]),
           dict(kept=w), dict(kept=tw), dict(kept=kept.pointer + 2), dict(kept=state), dict(kv_heads=0), dict(lengths=[64, 64]),
           dict(states=[state] * 2, contexts=[64] * 2, lengths=[64] * 2, weights=[w] * 2, targets=[target] * 2, target_contexts=[32] * 2, target_weights=[tw] * 2)]
    for change in bad:
        change = {k: [0 if x is None else x for x in v] if isinstance(v, list) else v for k, v in change.items()}
        with pytest.raises(StraydogError):
            gpu.kv8_evict(**{**good, **change})
    assert np.all(gpu.read(target, np.uint8, (state_bytes(32, 2, 64),)) == 0x22)
    for b in (state, target, w, tw, kept):
        gpu.release(b)
