"""8-bit K/V rows and masked attention at the ends of what they take, against the definition in 64 bits."""
import numpy as np
import pytest

from kv8_util import EPS, State, attention, evict, from_bits, rounded, state_bytes, to_bits
from test_gpu_kv8_attention import check

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
