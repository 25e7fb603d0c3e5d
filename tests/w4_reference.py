"""4-bit weights and the mixture-of-experts layer from their definitions, in 64 bits on the host, with bounds on what rounding may do to each result.

Bounds.  U = 2^-24 is half a step of fp32.  A sum of k products in fp32, in whatever order, is off by at most depth(k) * 2U * sum|terms|: depth is the longest
chain of additions that a term goes through, and matrix instructions may truncate where an addition rounds (hence 2U).  Terms go through one
instruction's 32 products, one chain over blocks of 32 k, and sums over wavefronts and lanes: depth(k) = 32 + k / 32 + 32.  bf16 weights are multiplied as
(128 + code) - (128 + zero), two products each, so there the terms' size is that of both.  A store to a type rounds by eps / 2 of the value."""
import numpy as np
import torch

U = 2.0 ** -24
TORCH = {0: torch.float32, 1: torch.float16, 3: torch.bfloat16}


def depth(k):
    return 64 + k / 32


def half_step(dtype):
    return torch.finfo(TORCH[dtype]).eps / 2


def smallest(dtype):
    """Half the distance of the smallest numbers of the type: what a rounding near zero may be off by."""
    f = torch.finfo(TORCH[dtype])
    return f.smallest_normal * f.eps / 2


def codes_of(q, k):
    """q: bytes [.., rows, bytes] -> codes [.., rows, k]."""
    q = q.numpy()
    return np.stack((q & 15, q >> 4), -1).reshape(q.shape[:-1] + (-1,))[..., :k].astype(np.float64)


class Weight:
    """Random 4-bit weights [.., rows, k] on the host: bytes, scales, zero points, and their values in 64 bits."""

    def __init__(self, g, dtype, rows, k, group, zeros=False, pad_bytes=0, pad_groups=0, lead=(), scale=0.05):
        self.k, self.group, self.groups = k, group, -(-k // group)
        self.q = torch.randint(0, 256, lead + (rows, (k + 1) // 2 + pad_bytes), generator=g, dtype=torch.uint8)
        self.scales = ((torch.rand(lead + (rows, self.groups + pad_groups), generator=g) + 0.5) * scale).to(TORCH[dtype])
        self.zeros = torch.randint(0, 16, lead + (rows, self.groups + pad_groups), generator=g, dtype=torch.uint8) if zeros else None
        self.ldq, self.lds = 2 * self.q.shape[-1], self.groups + pad_groups

    def spread(self, v):
        return np.repeat(v[..., :self.groups], self.group, -1)[..., :self.k]

    def parts(self):
        """(value, |code| + |zero| + 256 times the scale) in 64 bits."""
        s = self.spread(self.scales.double().numpy())
        z = self.spread(self.zeros.double().numpy()) if self.zeros is not None else 8.0
        c = codes_of(self.q, self.k)
        return (c - z) * s, (c + z + 256) * s


def gemm(dtype, w, b, alpha, beta, c):
    """(value, bound) of alpha * W * B + beta * C; b [n, k], c [n, m]."""
    b = b.double().numpy()
    value, size = w.parts()
    with np.errstate(invalid="ignore"):
        exact = alpha * (b @ value.T)
        terms = np.abs(b) @ (size if dtype == 3 else np.abs(value)).T
        if beta != 0:
            exact = exact + beta * c.double().numpy()
        # the products' sum, its product with the group's scale (a rounding for every group's sum), alpha, beta, the store
        off = abs(alpha) * (depth(w.k) + 4) * 2 * U * terms + 4 * U * np.abs(exact) + (2 * U * abs(beta) * np.abs(c.double().numpy()) if beta else 0)
        return exact, off + half_step(dtype) * (np.abs(exact) + off) + smallest(dtype)


def quantize(w, dtype, group, zeros):
    """(codes [m, k], scales [m, groups] in dtype, zeros or None): as the header defines them, in 64 bits."""
    top = torch.finfo(w.dtype).max
    v = torch.nan_to_num(w.double(), nan=0.0, posinf=top, neginf=-top).numpy()
    m, k = v.shape
    groups = -(-k // group)
    codes, scales, zs = np.zeros((m, k)), torch.zeros((m, groups), dtype=TORCH[dtype]), np.zeros((m, groups))
    for g in range(groups):
        part = v[:, g * group:(g + 1) * group]
        low, high = np.minimum(part.min(1), 0), np.maximum(part.max(1), 0)
        s = (high - low) / 15 if zeros else np.maximum(high, -low) / 7
        s = torch.from_numpy(s.astype(np.float32)).clamp(max=torch.finfo(TORCH[dtype]).max).to(TORCH[dtype])
        scales[:, g] = s
        s = s.double().numpy()
        safe = np.where(s == 0, 1, s)
        z = np.clip(np.rint(-low / safe), 0, 15) if zeros else np.full(m, 8.0)
        z = np.where(s == 0, 0 if zeros else 8, z)
        zs[:, g] = z
        codes[:, g * group:(g + 1) * group] = np.where(s[:, None] == 0, z[:, None], np.clip(np.rint(part / safe[:, None]) + z[:, None], 0, 15))
    return codes, scales, zs if zeros else None


def select(logits, top_k, sigmoid, renormalize, bias):
    """(ids, weights) of each token from logits [t, e] in 64 bits."""
    with np.errstate(all="ignore"):
        score = 1 / (1 + np.exp(-logits)) if sigmoid else np.exp(logits - np.nanmax(logits, 1, keepdims=True))
        if not sigmoid:
            score = score / score.sum(1, keepdims=True)
        key = logits if bias is None else score + bias
        key = np.where(np.isnan(key), -np.inf, key)
        ids = np.argsort(-key, axis=1, kind="stable")[:, :top_k]
        w = np.take_along_axis(score, ids, 1)
        if renormalize:
            total = w.sum(1, keepdims=True)
            w = np.where(total == 0, 0, w / np.where(total == 0, 1, total))
    return ids, w


def moe(dtype, x, router, gate_up, down, inner, top_k, sigmoid=False, renormalize=True, bias=None, alpha=1.0, beta=0.0, y=None):
    """(value, bound, ids, weights).  x, y [t, h]; router [e, h]; gate_up, down: Weight or 16-bit tensors [e, rows, k]."""
    x64 = x.double().numpy()
    t, h = x64.shape
    ids, weights = select(x64 @ router.double().numpy().T, top_k, sigmoid, renormalize, None if bias is None else bias.double().numpy())

    def parts(w, e):
        if isinstance(w, torch.Tensor):
            v = w[e].double().numpy()
            return v, np.abs(v)
        one = object.__new__(Weight)
        one.__dict__.update(w.__dict__, q=w.q[e], scales=w.scales[e], zeros=None if w.zeros is None else w.zeros[e])
        value, size = one.parts()
        return value, size if dtype == 3 else np.abs(value)

    value, off = np.zeros((t, h)), np.zeros((t, h))
    for e in np.unique(ids):
        a, s = np.nonzero(ids == e)
        (w1, t1), (w2, t2) = parts(gate_up, e), parts(down, e)
        gu, terms = x64[a] @ w1.T, (depth(h) + 4) * 2 * U * (np.abs(x64[a]) @ t1.T)
        g, u, dg, du = gu[:, :inner], gu[:, inner:], terms[:, :inner], terms[:, inner:]
        with np.errstate(over="ignore"):
            silu = g / (1 + np.exp(-g))
        # |silu'| < 1.1; exp, the quotient and the product: 8 half steps; h as two numbers of the type: half a step of the second one
        hv = silu * u
        dh = 1.1 * dg * np.abs(u) + np.abs(silu) * du + 1.1 * dg * du + 16 * U * np.abs(hv) + half_step(dtype) ** 2 * np.abs(hv) + smallest(dtype)
        wt = weights[a, s][:, None]
        value[a] += wt * (hv @ w2.T)
        off[a] += np.abs(wt) * (dh @ np.abs(w2).T + (depth(inner) + top_k + 4) * 2 * U * ((np.abs(hv) + dh) @ t2.T))
    exact = alpha * value + (beta * y.double().numpy() if beta else 0)
    off = abs(alpha) * off + 4 * U * np.abs(exact) + (2 * U * abs(beta) * np.abs(y.double().numpy()) if beta else 0)
    return exact, off + half_step(dtype) * (np.abs(exact) + off) + smallest(dtype), ids, weights
