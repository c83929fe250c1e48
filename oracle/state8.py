"""The 8-bit optimizer state in numpy, from its definition (include/elx_ops.h), and the Adam step over it: decode, the fp32
step of the C oracle, encode.  Test infrastructure."""
import numpy as np
import torch

from . import oracle as O

BLOCK = 256
HALF = 1 << 19
_U32 = np.uint32


def mix(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, dtype=_U32)
    with np.errstate(over='ignore'):
        x = (x ^ (x >> _U32(16))) * _U32(0x6A09E667)
        x = (x ^ (x >> _U32(15))) * _U32(0xBB67AE85)
    return x ^ (x >> _U32(16))


def dither(blocks: np.ndarray, salt: int, step: int) -> np.ndarray:
    """[len(blocks), 256] values of 20 bits."""
    with np.errstate(over='ignore'):
        seed = mix(np.array([(salt * 0x9E3779B9 + step) & 0xFFFFFFFF], dtype=_U32))
        key = mix(np.asarray(blocks, dtype=_U32) ^ seed)
        lane = np.arange(64, dtype=_U32) * _U32(0x9E3779B9)
        word = mix(key[:, None] + lane[None, :]).astype(np.uint64)
    turn = np.arange(4, dtype=np.uint64) * np.uint64(8)
    turned = ((word[..., None] >> turn) | (word[..., None] << (np.uint64(32) - turn))) & np.uint64(0xFFFFFFFF)
    return (turned >> np.uint64(12)).astype(np.int64).reshape(len(blocks), BLOCK)


def to_blocks(x: np.ndarray) -> np.ndarray:
    out = np.zeros((-(-x.size // BLOCK), BLOCK), dtype=x.dtype)
    out.reshape(-1)[:x.size] = x
    return out


def exponent(x: np.ndarray) -> np.ndarray:
    """E of every block of fp32 values [blocks, 256]: the smallest with max <= 1.75 * 2^(E - 127) over the finite ones
    (0 up to 1.5 * 2^-127)."""
    top = np.where(np.isfinite(x), np.abs(x), 0).max(axis=1).astype(np.float64)
    e = np.zeros(len(top), dtype=np.int64)
    some = top > 0
    f, p = np.frexp(top[some])
    e[some] = np.maximum(1, p - 1 + 127 + (f > 0.875))
    return np.where(top > 1.5 * 2.0**-127, e, 0)


def encode_avg(x: np.ndarray):
    """fp32 [blocks, 256] -> (codes uint8, E): nearest even."""
    e = exponent(x)
    scaled = np.ldexp(x, (135 - e)[:, None].astype(np.int32)).astype(np.float32)
    codes = torch.from_numpy(scaled).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    over = (e == 255)[:, None] & ((codes & 0x7F) > 0x77)    # 2^128: the largest value of fp32 is below
    codes = np.where(over, (codes & 0x80) | 0x77, codes)
    return np.where(np.isfinite(x), codes, 0x7F).astype(np.uint8), e


def encode_sq(x: np.ndarray, r: np.ndarray):
    """fp32 [blocks, 256] and 20 bits each -> (codes uint8, E)."""
    e = exponent(x)
    bits = np.ldexp(x, (31 - e)[:, None].astype(np.int32)).astype(np.float32).view(np.uint32).astype(np.int64)
    codes = np.maximum((bits + r) >> 20, (x != 0).astype(np.int64))
    codes = np.where((e == 255)[:, None], np.minimum(codes & 0xFF, 0xF7), codes)
    return np.where(np.isfinite(x), codes, 0xFF).astype(np.uint8), e


def decode_avg(codes: np.ndarray, e: np.ndarray) -> np.ndarray:
    c = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).to(torch.float32).numpy()
    return np.ldexp(c, (np.asarray(e, dtype=np.int64) - 135)[:, None].astype(np.int32)).astype(np.float32)


def decode_sq(codes: np.ndarray, e: np.ndarray) -> np.ndarray:
    v = (codes.astype(np.uint32) << _U32(20)).view(np.float32)
    v = np.ldexp(v, (np.asarray(e, dtype=np.int64) - 31)[:, None].astype(np.int32)).astype(np.float32)
    return np.where(codes == 0xFF, np.float32(np.nan), v)


class State8:
    """The 8-bit moments of one flat buffer of n elements."""

    def __init__(self, n: int, salt: int = 0):
        self.n, self.salt = n, salt
        blocks = -(-n // BLOCK)
        self.m, self.v = np.zeros((blocks, BLOCK), np.uint8), np.zeros((blocks, BLOCK), np.uint8)
        self.me, self.ve = np.zeros(blocks, np.int64), np.zeros(blocks, np.int64)

    def set(self, m: np.ndarray, v: np.ndarray) -> None:
        self.m, self.me = encode_avg(to_blocks(m.astype(np.float32)))
        self.v, self.ve = encode_sq(to_blocks(v.astype(np.float32)), HALF)

    def values(self):
        return (decode_avg(self.m, self.me).reshape(-1)[:self.n].copy(), decode_sq(self.v, self.ve).reshape(-1)[:self.n].copy())

    def step(self, p: np.ndarray, g, g_dtype: int, segments=None, **hyper) -> None:
        """One step of fp32 ``p`` in place.  ``segments``: [(begin, end, hyper keywords)] (default: all of it with
        ``hyper``); blocks no segment touches keep their bits."""
        segments = [(0, self.n, {})] if segments is None else segments
        m, v = self.values()
        r = np.full((len(self.me), BLOCK), HALF, dtype=np.int64)
        touched = np.zeros(len(self.me), dtype=bool)
        every = np.arange(len(self.me))
        for begin, end, more in segments:
            kw = dict(hyper, **more)
            ps, ms, vs = p[begin:end].copy(), m[begin:end].copy(), v[begin:end].copy()
            O.adam(None if g is None else g[begin:end].copy(), g_dtype, ps, ms, vs, **kw)
            p[begin:end], m[begin:end], v[begin:end] = ps, ms, vs
            r.reshape(-1)[begin:end] = dither(every, self.salt, kw['step'] & 0xFFFFFF).reshape(-1)[begin:end]
            touched[begin // BLOCK:-(-end // BLOCK)] = True
        mc, me = encode_avg(to_blocks(m))
        vc, ve = encode_sq(to_blocks(v), r)
        self.m[touched], self.me[touched] = mc[touched], me[touched]
        self.v[touched], self.ve[touched] = vc[touched], ve[touched]
        tail = len(self.me) * BLOCK - self.n    # what lies behind the last element does not exist
        if tail:
            self.m[-1, -tail:] = 0
            self.v[-1, -tail:] = 0
