"""sdx_masked_attention (packed documents over 16-bit keys and values; caps, distance biases, windows, prefixes) against the definition in 64 bits."""
import numpy as np
import pytest

from kv8_util import attention, from_bits, to_bits, tolerance

pytestmark = pytest.mark.gpu
GUARD = 64


def attend(gpu, q, k, v, rows, lengths, kind, fused=False, out_pad=0, **rule):
    """q [total][heads][dim], k and v [keys][kv_heads][dim] float32. fused: parts of one array's rows."""
    (total, heads, dim), (keys, kv_heads, _) = q.shape, k.shape
    (qr, qh), (kr, kh), (vr, vh) = (to_bits(x, kind) for x in (q, k, v))
    strides = {}
    if fused:
        one = np.concatenate([x.reshape(total, -1) for x in (qr, kr, vr)] + [np.full((total, 8), 0x7fff, np.int16)], 1)
        buffers = [gpu.upload(one)]
        at = [buffers[0].at(0), buffers[0].at(heads * dim * 2), buffers[0].at((heads + kv_heads) * dim * 2)]
        strides = dict(q_stride=one.shape[1], k_stride=one.shape[1], v_stride=one.shape[1])
    else:
        buffers = [gpu.upload(x) for x in (qr, kr, vr)]
        at = [b.pointer for b in buffers]
    width = heads * dim
    out = gpu.upload(np.full(total * (width + out_pad) + GUARD, 0x5a5a, np.int16))
    slopes = rule.pop("slopes", None)
    if slopes is not None:
        buffers.append(gpu.upload(np.asarray(slopes, np.float32)))
        rule["slopes"] = buffers[-1]
    gpu.masked_attention(*at, out, rows, lengths, heads, kv_heads, dim, kind, dim ** -0.5, out_stride=width + out_pad, **strides, **rule)
    got = gpu.read(out, np.int16, (total * (width + out_pad) + GUARD,))
    assert gpu.decode_status() == 0
    got, guard = got[:-GUARD].reshape(total, width + out_pad), got[-GUARD:]
    assert np.all(guard == 0x5a5a) and np.all(got[:, width:] == 0x5a5a), "what lies beside the output"
    for b in buffers + [out]:
        gpu.release(b)
    return from_bits(np.ascontiguousarray(got[:, :width]), kind).reshape(total, heads, dim), qh, kh, vh


def check(gpu, rows, lengths, heads, kv_heads, dim, kind, seed, prefixes=None, spoil=None, **rule):
    rng = np.random.default_rng(seed)
    q = rng.normal(size=(sum(rows), heads, dim)).astype(np.float32)
    k, v = (rng.normal(size=(sum(lengths), kv_heads, dim)).astype(np.float32) for _ in range(2))
    if spoil:
        spoil(q, k, v)
    extra = {"prefixes": prefixes} if prefixes else {}
    got, qh, kh, vh = attend(gpu, q, k, v, rows, lengths, kind, **extra, **rule)
    rule = {name: value for name, value in rule.items() if name not in ("fused", "out_pad")}
    row = key = 0
    for d, (r, n) in enumerate(zip(rows, lengths)):
        with np.errstate(invalid="ignore"):
            want, _, size = attention(qh[row:row + r], kh[key:key + n], vh[key:key + n], dim ** -0.5, prefix=prefixes[d] if prefixes else 0, **rule)
        mine = got[row:row + r]
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(mine), np.isnan(want)) and np.array_equal(mine[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), d
        off = np.abs(mine - want)[fine]
        bound = tolerance(kind, want, size)[fine]
        assert np.all(off <= bound), (d, r, n, float((off / bound).max()))
        row, key = row + r, key + n


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (64, 7, 1), (128, 8, 2), (128, 24, 2), (256, 4, 2), (256, 16, 1)])
def test_ragged_documents(gpu, kind, dim, heads, kv_heads):
    rows, lengths = [1, 130, 0, 77, 5, 300, 9], [1, 130, 4, 500, 0, 300, 3]   # (no rows, no keys, fewer keys than rows)
    check(gpu, rows, lengths, heads, kv_heads, dim, kind, dim + heads)


@pytest.mark.parametrize("rule", [dict(cap=2.0), dict(slopes=True), dict(window=1), dict(window=100), dict(prefixes=[129, 0, 40]), dict(prefixes=[400, 200, 128]),
                                  dict(window=64, prefixes=[1, 150, 128]), dict(cap=4.0, slopes=True, window=130, prefixes=[7, 0, 128])], ids=lambda r: "-".join(r))
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 6, 2), (128, 4, 1), (256, 6, 3)])
def test_rules(gpu, rule, dim, heads, kv_heads):
    rule = dict(rule)
    if rule.pop("slopes", None):
        rule["slopes"] = np.exp2(-np.arange(1, heads + 1) / 2).astype(np.float32)
    check(gpu, [260, 200, 50], [400, 200, 128], heads, kv_heads, dim, 30 if dim == 128 else 1, dim, **rule)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_parts_of_one_projections_rows_and_a_wider_output(gpu, dim):
    check(gpu, [200, 33], [200, 33], 4, 2, dim, 30, dim, fused=True, out_pad=16)


@pytest.mark.parametrize("dim,rows,length", [(64, 3, 9000), (128, 100, 5000), (256, 1, 7000), (256, 64, 3000)])
def test_few_rows_over_many_keys(gpu, dim, rows, length):
    # (the key range is cut over several blocks)
    check(gpu, [rows], [length], 4, 1, dim, 1, dim + rows)
    check(gpu, [rows, 2], [length, 2000], 4, 2, dim, 30, dim + rows, window=1500, prefixes=[200, 0])


def test_more_documents_than_a_launch_takes(gpu):
    rows = [1 + 7 * d % 23 for d in range(150)]
    check(gpu, rows, rows, 2, 2, 64, 1, 3)


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, kind, dim):
    # infinities and NaN in the keys and values of later positions, of other documents, of what the window has left; a row that sees them
    # has them: a value's column, a key's whole row
    def spoil(q, k, v):
        v[150, 0, 3], v[151, 1, 5], v[300, 0, :] = np.nan, np.inf, -np.inf   # (document 0 has 200 keys, document 1 150)
        v[349, 1, 60] = np.nan
        k[360, 0, 2], k[361, 1, 1] = np.nan, np.inf
    check(gpu, [200, 150, 100], [200, 150, 100], 4, 2, dim, kind, 5, spoil=spoil)
    check(gpu, [200, 150, 100], [200, 150, 100], 4, 2, dim, kind, 6, spoil=spoil, window=20, prefixes=[0, 130, 0])


def test_a_nan_query_row_stays_its_own(gpu):
    def spoil(q, k, v):
        q[40, 1, 3], q[41, 0, 0] = np.nan, np.inf
    rng = np.random.default_rng(4)
    q = rng.normal(size=(90, 2, 128)).astype(np.float32)
    k, v = (rng.normal(size=(90, 2, 128)).astype(np.float32) for _ in range(2))
    clean, _, _, _ = attend(gpu, q, k, v, [90], [90], 30)
    spoil(q, k, v)
    got, _, _, _ = attend(gpu, q, k, v, [90], [90], 30)
    assert np.all(np.isnan(got[40, 1])) and np.all(np.isnan(got[41, 0]))
    got[40, 1], got[41, 0] = clean[40, 1], clean[41, 0]
    assert np.array_equal(got, clean)


def test_large_scores(gpu):
    # scores of a few hundred: all weight on one key, the maximum moves often
    def spoil(q, k, v):
        q *= 30
        k *= 4
    for dim in (64, 128, 256):
        check(gpu, [300], [300], 2, 1, dim, 1, 9, spoil=spoil, cap=200.0)


def test_refusals(gpu):
    from straydog_b200.backend import StraydogError
    q, k, v = gpu.buffer(8 * 4 * 64 * 2), gpu.buffer(8 * 2 * 64 * 2), gpu.buffer(8 * 2 * 64 * 2)
    out = gpu.upload(np.full(8 * 4 * 64, 0x5a5a, np.int16))
    good = dict(q=q.pointer, k=k.pointer, v=v.pointer, out=out.pointer, rows=[8], lengths=[8], heads=4, kv_heads=2, dim=64, type=1, scale=0.1)
    bad = [dict(heads=3), dict(kv_heads=0), dict(dim=32), dict(type=0), dict(type=24), dict(scale=-1.0), dict(cap=float("nan")), dict(rows=[9]), dict(lengths=[9]),
           dict(q_stride=248), dict(k_stride=132), dict(v_stride=120), dict(q=q.pointer + 8), dict(k=None), dict(out=q.pointer), dict(out=k.pointer, heads=2),
           dict(slopes=4), dict(rows=[2 ** 33]), dict(lengths=[2 ** 33]), dict(rows=[8, 1]), dict(prefixes=[1, 1]), dict(heads=516, kv_heads=4), dict(rows=[], lengths=[])]
    for change in bad:
        with pytest.raises(StraydogError):
            gpu.masked_attention(**{**good, **change})
    assert np.all(gpu.read(out, np.int16, (8 * 4 * 64,)) == 0x5a5a)
    gpu.masked_attention(**{**good, "rows": [0]})
    assert np.all(gpu.read(out, np.int16, (8 * 4 * 64,)) == 0x5a5a)
    for b in (q, k, v, out):
        gpu.release(b)


@pytest.mark.parametrize("kind", [1, 30])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 1), (128, 4, 2), (256, 4, 1)])
@pytest.mark.parametrize("cap,size", [(0.0, 1.0), (5.0, 0.5), (50.0, 1.0), (50.0, 20.0)])
def test_caps_and_biases_over_many_tiles(gpu, kind, dim, heads, kv_heads, cap, size):
    # slopes of either sign from flat to steep, keys behind, across and ahead of the rows (a prefix past them), scores within and far past the cap's series
    def spoil(q, k, v):
        q *= np.float32(size)

    slopes = np.asarray([0.0, 0.004, 0.06, 0.7, -0.003, 0.02, 0.25, -0.0001], np.float32)[:heads]
    check(gpu, [260, 700, 130], [900, 700, 1100], heads, kv_heads, dim, kind, dim + heads, cap=cap, slopes=slopes, spoil=spoil)
    check(gpu, [300, 200], [700, 900], heads, kv_heads, dim, kind, dim, prefixes=[640, 900], cap=cap, slopes=slopes, spoil=spoil)
    check(gpu, [300], [800], heads, kv_heads, dim, kind, dim + 1, cap=cap, window=333, slopes=-slopes, spoil=spoil)
    check(gpu, [600], [600], heads, kv_heads, dim, kind, dim + 2, cap=cap, spoil=spoil)
