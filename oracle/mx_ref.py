"""TEST INFRASTRUCTURE -- microscaled storage in float64 (numpy), from the format's definition: 32 consecutive channels share a power-of-two scale, the
elements are E4M3 or E2M1 codes.  Plain loops over tables; never imported by the product."""
import numpy as np

CODES = {'e2m1': [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
         'e4m3': [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]}
TOP_FRACTION = {'e2m1': 1.5, 'e4m3': 1.875}      # of the type's largest power of two: the largest magnitude kept
TYPE_EXPONENT = {'fp16': 15, 'bf16': 127, 'fp32': 127}
MIN_SCALE, NAN_SCALE = 10, 255


def pack(x, dtype, fmt):
    """x float64 [rows, C], every value one of `dtype` ('fp32', 'bf16', 'fp16') -> codes uint8 [rows, nb * 32 or 16], scales uint8 [rows, nb]"""
    table = np.array(CODES[fmt])
    rows, c = x.shape
    nb = (c + 31) // 32
    v = np.zeros((rows, nb * 32))
    v[:, :c] = x
    v = v.reshape(rows, nb, 32)
    fine = np.isfinite(v).all(2)
    lim = TOP_FRACTION[fmt] * 2.0 ** TYPE_EXPONENT[dtype]
    v = np.clip(np.where(fine[:, :, None], v, 0.0), -lim, lim)
    amax = np.abs(v).max(2)
    man, ex = np.frexp(amax / table[-1])
    ex = np.where(man == 0.5, ex - 1, ex)
    byte = np.maximum(np.where(amax == 0, -1000, ex) + 127, MIN_SCALE)
    a = np.ldexp(np.abs(v), 127 - byte[:, :, None])
    mids = (table[1:] + table[:-1]) / 2
    at = np.searchsorted(mids, a, side='left')
    tie = (at < len(mids)) & (a == mids[np.minimum(at, len(mids) - 1)])
    at = at + (tie & (at % 2 == 1))                                        # the even code of the two
    half = 128 if fmt == 'e4m3' else 8
    code = np.where(fine[:, :, None], at + half * np.signbit(v), 0).reshape(rows, nb * 32)
    if fmt == 'e2m1':
        code = code[:, 0::2] + 16 * code[:, 1::2]
    return code.astype(np.uint8), np.where(fine, byte, NAN_SCALE).astype(np.uint8)


def unpack(codes, scales, c, fmt):
    """the values, float64 [rows, c]"""
    table = np.array(CODES[fmt])
    k = codes.astype(np.int64)
    if fmt == 'e2m1':
        k = np.stack([k % 16, k // 16], 2).reshape(k.shape[0], -1)
    half = 128 if fmt == 'e4m3' else 8
    v = np.append(table, np.nan)[k % half] * np.where(k >= half, -1.0, 1.0) if fmt == 'e4m3' else table[k % half] * np.where(k >= half, -1.0, 1.0)
    s = np.where(scales == NAN_SCALE, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(k.shape[0], -1, 32) * s[:, :, None]).reshape(k.shape[0], -1)[:, :c]


def conv_weight_grad(dy, x, kh, kw, stride, pad):
    """dy [N,H,W,A], x [N,Hi,Wi,B] float64 -> (gradient, sum of the absolute products), both [A,kh,kw,B]"""
    n, h, w, a = dy.shape
    g, s = np.zeros((a, kh, kw, x.shape[3])), np.zeros((a, kh, kw, x.shape[3]))
    for i in range(kh):
        for j in range(kw):
            for y in range(h):
                for z in range(w):
                    iy, ix = y * stride - pad + i, z * stride - pad + j
                    if 0 <= iy < x.shape[1] and 0 <= ix < x.shape[2]:
                        g[:, i, j] += dy[:, y, z].T @ x[:, iy, ix]
                        s[:, i, j] += np.abs(dy[:, y, z]).T @ np.abs(x[:, iy, ix])
    return g, s


def batchnorm_forward(y, gamma, beta, eps):
    mean, var = y.mean(0), y.var(0)
    invstd = 1 / np.sqrt(var + eps)
    return (y - mean) * invstd * gamma + beta, mean, invstd


def batchnorm_backward(dout, y, gamma, mean, invstd, mask=None):
    """dy, dgamma, dbeta, dh of float64 [rows, C]"""
    dh = dout if mask is None else np.where(mask, dout, 0.0)
    xhat = (y - mean) * invstd
    dbeta, dgamma = dh.sum(0), (dh * xhat).sum(0)
    n = y.shape[0]
    return gamma * invstd * (dh - dbeta / n - xhat * dgamma / n), dgamma, dbeta, dh
