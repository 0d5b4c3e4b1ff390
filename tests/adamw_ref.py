"""One AdamW step in 64 bits (parameters, fp32 states) and, for states in 8 bits, in fp32 with every operation rounded by itself, as the
definition has it: the codes are then equal bit for bit."""
import numpy as np

F = np.float32
BLOCK = 128


def mix(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x7FEB352D)) & np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0x846CA68B)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def word(seed, t, i):
    h = mix((seed ^ (20 * 0x9E3779B9)) & 0xFFFFFFFF)
    h = mix(int(h) ^ ((t * 0x85EBCA6B + 0x165667B1) & 0xFFFFFFFF))
    i = np.asarray(i, np.uint64)
    h = mix(h ^ (((i >> np.uint64(32)) * np.uint64(0xC2B2AE35) + np.uint64(0x27D4EB2F)) & np.uint64(0xFFFFFFFF)))
    return mix(h ^ (((i & np.uint64(0xFFFFFFFF)) * np.uint64(0x9E3779B1) + np.uint64(0x85EBCA77)) & np.uint64(0xFFFFFFFF)))


def e4m3(code):
    """The value of an e4m3 byte (no NaN: the largest code that occurs is below 256)."""
    code = np.asarray(code, np.uint8).astype(np.int64)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    return np.where(code & 0x80, -v, v)


def decode(code, scale):
    with np.errstate(over="ignore"):
        s = np.where(scale == 255, np.nan, 2.0 ** (np.asarray(scale, np.float64) - 127))
    return (e4m3(code).reshape(-1, BLOCK) * s[:, None]).reshape(-1)


def encode(x, w16, positive):
    """x fp32 [blocks * 128], w16: 16 random bits each -> codes, scale bytes."""
    x = np.asarray(x, F)
    top = np.abs(x).view(np.uint32).reshape(-1, BLOCK).max(1)
    e = (top >> 23).astype(np.int64)
    scale = np.where(e == 255, 255, np.maximum(e - 7, 16))
    with np.errstate(under="ignore", invalid="ignore"):
        y = (np.abs(x).astype(np.float64).reshape(-1, BLOCK) * 2.0 ** (7.0 - scale[:, None])).astype(F).view(np.uint32).astype(np.uint64).reshape(-1)
    code = (y + (np.asarray(w16, np.uint64) << np.uint64(4)) + np.uint64(8)) >> np.uint64(20)
    if positive:
        code = np.where((x > 0) & (code == 0), np.uint64(1), code)
    else:
        code = code | ((x.view(np.uint32) >> 24) & 0x80).astype(np.uint64)
    code = np.where(np.repeat(e == 255, BLOCK), np.uint64(0), code)
    return code.astype(np.uint8), scale.astype(np.uint8)


def factor(grads, clip, grad_scale):
    norm = grad_scale * np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads))
    return norm, (grad_scale * (clip / max(norm, clip)) if clip > 0 else grad_scale)


def step64(p, g, m, v, t, gs, lr, b1, b2, eps, decay):
    """float64 arrays; returns p, m, v and bounds of what fp32 may be off (u = 2^-24): m, v: products, sums and the rounded gs; p: the
    kept part rounded twice, the update's factors, root and reciprocal (one ulp each) and the errors of m and v in it."""
    u = 2.0 ** -24
    x = gs * g
    mn, vn = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    em = 4 * u * (np.abs(b1 * m) + np.abs((1 - b1) * x)) + 2.0 ** -149
    ev = 6 * u * vn + 2.0 ** -148
    lt, c = lr / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    den = np.sqrt(vn) * c + eps
    upd = lt * mn / den
    # a root next to nothing: |sqrt(v + e) - sqrt(v)| <= sqrt(e)
    er = np.minimum(np.sqrt(ev), ev / np.maximum(np.sqrt(vn), 1e-300)) * c
    pn = p * (1 - lr * decay) - upd
    ep = 3 * u * np.abs(p) + lt * em / den + np.abs(upd) * (16 * u + er / den) + u * np.abs(pn)
    return pn, mn, vn, ep, em, ev


def step8(m8, ms, v8, vs, g, t, gs, b1, b2, seed, at):
    """Codes and scales behind a step; g fp32, m8 ... whole blocks, at: index of the first element in the state buffers.  Also the
    unrounded m and v (fp32)."""
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        m, r = decode(m8, ms).astype(F), decode(v8, vs).astype(F)
        x = g.astype(F) * F(gs)
        mn = m * F(b1) + x * F(1 - b1)
        vn = (r * r) * F(b2) + (x * x) * F(1 - b2)
        rn = np.sqrt(vn)
    w = word(seed, t, at + np.arange(m.size))
    return encode(mn, w & np.uint64(0xFFFF), False) + encode(rn, w >> np.uint64(16), True) + (m, r)
