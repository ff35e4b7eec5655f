"""The definition of the 8-bit rows with block scales, of the masked attention and of the eviction, in numpy (64 bits where values are computed)."""
import numpy as np
import torch

BLOCK = 32
TOP = {0: 127.0, 1: 448.0}
TYPES = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
EPS = {1: 2.0 ** -11, 30: 2.0 ** -8}   # half a step of an output, relative (F16, BF16)


def rounded(context):
    return -(-context // BLOCK) * BLOCK


def state_bytes(context, kv_heads, dim):
    return -(-2 * kv_heads * (context * dim + context // BLOCK * 4) // 16) * 16


def to_bits(x, kind):
    """float32 numpy -> (the bytes of that type, the values they hold as float64)"""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TYPES[kind])
    raw = t.view(torch.int32 if kind == 0 else torch.int16).numpy()
    return raw, t.double().numpy()


def from_bits(raw, kind):
    return torch.from_numpy(raw).view(TYPES[kind]).double().numpy()


def encode(y, code):
    """float32 quotients -> (codes as uint8)"""
    y = torch.from_numpy(np.ascontiguousarray(y, np.float32))
    if code == 0:
        return torch.round(y.nan_to_num(nan=0.0, posinf=127, neginf=-127)).clamp(-127, 127).to(torch.int8).numpy().view(np.uint8)
    return y.nan_to_num(nan=0.0, posinf=448, neginf=-448).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def decode(raw, code):
    raw = np.ascontiguousarray(raw)
    if code == 0:
        return raw.view(np.int8).astype(np.float32)
    return torch.from_numpy(raw).view(torch.float8_e4m3fn).float().numpy()


class State:
    """A state in host memory: codes [planes][context][dim] and scales [planes][context / 32]."""

    def __init__(self, context, kv_heads, dim, code, fill=0):
        self.context, self.kv_heads, self.dim, self.code = context, kv_heads, dim, code
        self.codes = np.full((2 * kv_heads, context, dim), fill, np.uint8)
        self.scales = np.zeros((2 * kv_heads, context // BLOCK), np.float32)

    def write(self, base, keys, values):
        """keys, values: [steps][kv_heads][dim] float32, the definition step by step in float32"""
        steps = keys.shape[0]
        rows = np.concatenate([keys, values], 1).transpose(1, 0, 2).astype(np.float32)
        for plane in range(2 * self.kv_heads):
            for block in range(base // BLOCK, (base + steps - 1) // BLOCK + 1):
                begin = block * BLOCK
                low, high = max(begin, base), min(begin + BLOCK, base + steps)
                x = rows[plane, low - base:high - base]
                finite = np.where(np.isfinite(x), np.abs(x), np.float32(0))
                need = np.float32(finite.max()) / np.float32(TOP[self.code])
                old = self.scales[plane, block] if begin < base else np.float32(0)
                scale = max(old, need)
                if begin < base and scale > old:
                    ratio = np.float32(old) / np.float32(scale)
                    self.codes[plane, begin:low] = encode(decode(self.codes[plane, begin:low], self.code) * ratio, self.code)
                with np.errstate(all="ignore"):
                    self.codes[plane, low:high] = encode(x / scale, self.code) if scale > 0 else 0
                self.scales[plane, block] = scale
        return self

    def pack(self):
        raw = np.concatenate([self.codes.reshape(-1), self.scales.reshape(-1).view(np.uint8)])
        return np.concatenate([raw, np.zeros(state_bytes(self.context, self.kv_heads, self.dim) - raw.size, np.uint8)])

    def unpack(self, raw):
        n = self.codes.size
        other = State(self.context, self.kv_heads, self.dim, self.code)
        other.codes = raw[:n].reshape(self.codes.shape).copy()
        other.scales = raw[n:n + self.scales.size * 4].view(np.float32).reshape(self.scales.shape).copy()
        return other

    def values(self, length):
        """([length][kv_heads][dim] keys, values) as float64"""
        v = decode(self.codes[:, :length], self.code).astype(np.float64) * np.repeat(self.scales, BLOCK, 1)[:, :length, None].astype(np.float64)
        return v[:self.kv_heads].transpose(1, 0, 2), v[self.kv_heads:].transpose(1, 0, 2)


def random_state(rng, context, kv_heads, dim, code, length, spread=1.0):
    """A state whose first `length` rows hold normal values, block sizes spread over powers of two"""
    state = State(context, kv_heads, dim, code, fill=0x55)
    if length:
        x = rng.normal(size=(2, length, kv_heads, dim)).astype(np.float32)
        x *= np.exp2(spread * rng.normal(size=(2, length, 1, 1))).astype(np.float32)
        state.write(0, x[0], x[1])
    return state


def seen(rows, length, window=0, prefix=0):
    p, j = np.arange(rows)[:, None] + (length - rows), np.arange(length)[None, :]
    mask = j <= p
    if window:
        mask = mask & (j > p - window)
    return mask | (j < prefix)


def attention(q, k, v, scale, cap=0.0, slopes=None, window=0, prefix=0):
    """q [rows][heads][dim], k and v [length][kv_heads][dim], float64: (out, weights [kv_heads][length], the sums of |p v|)"""
    rows, heads, dim = q.shape
    length, kv_heads = k.shape[:2]
    out, size, weights = np.zeros_like(q), np.zeros_like(q), np.zeros((kv_heads, length))
    mask = seen(rows, length, window, prefix)
    distance = np.abs(np.arange(rows)[:, None] + (length - rows) - np.arange(length)[None, :])
    for h in range(heads):
        kv = h // (heads // kv_heads)
        s = q[:, h] @ np.where(mask.any(0)[:, None], k[:, kv], 0.0).T * scale if length else np.zeros((rows, 0))
        if cap:
            s = cap * np.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * distance
        s = np.where(mask, s, -np.inf)
        top = np.where(mask.any(1), s.max(1, initial=-np.inf), 0.0)
        p = np.exp(s - top[:, None])
        total = p.sum(1)
        p = p / np.where(total > 0, total, 1.0)[:, None]
        for i in range(rows):   # (a masked value is not multiplied: it may be infinite)
            at = mask[i]
            out[i, h] = p[i, at] @ v[at, kv]
            size[i, h] = p[i, at] @ np.abs(v[at, kv])
        weights[kv] += p.sum(0)
    return out, weights, size


def evict(state, length, weights, keep, sinks, recent):
    """(target State of rounded(keep) positions, kept [kv_heads][count], their weights)"""
    target = State(rounded(keep), state.kv_heads, state.dim, state.code)
    count = min(length, keep)
    kept = np.zeros((state.kv_heads, count), np.int64)
    for h in range(state.kv_heads):
        if length <= keep:
            kept[h] = np.arange(length)
            continue
        middle = np.arange(sinks, length - recent)
        w = weights[h, middle].astype(np.float64)
        order = np.lexsort((middle, -np.where(np.isnan(w), 0.0, w), np.isnan(w)))
        chosen = middle[order[:keep - sinks - recent]]
        kept[h] = np.sort(np.concatenate([np.arange(sinks), chosen, np.arange(length - recent, length)]))
    for plane in range(2 * state.kv_heads):
        at = kept[plane % state.kv_heads]
        for block in range(-(-count // BLOCK)):
            rows = at[block * BLOCK:(block + 1) * BLOCK]
            old = state.scales[plane, rows // BLOCK]
            scale = old.max()
            ratio = old / scale if scale > 0 else np.zeros_like(old)
            target.codes[plane, block * BLOCK:block * BLOCK + rows.size] = encode(decode(state.codes[plane, rows], state.code) * ratio[:, None], state.code)
            target.scales[plane, block] = scale
    return target, kept, np.take_along_axis(weights, kept, 1)


def tolerance(kind, out, size):
    """What an output may be off: its own rounding (half a step of |out|), the weights' rounding on their way to the tensor cores (FP16 or BF16 by
    the rows' type, half a step of each weight: at most that of the sum of |p v|), and 2^-16 of that sum for the FP32 scores, sums and exponentials
    (scores of up to 2^6 at 2^-24 each, 2^-22 an exponential, sums of up to 2^6 roundings)."""
    return EPS[kind] * np.abs(out) + (EPS[kind] + 2.0 ** -16) * size + 1e-7
