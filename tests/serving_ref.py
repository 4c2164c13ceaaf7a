"""Plain float64 forms of the serving operators, row by row, and the error
bounds that their tests use."""
import math

import numpy as np
import torch

NO_PAGE = 0xFFFFFFFF
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.uint32)).view(np.int32)).cuda()


class Case:
    """A ragged batch with random pages: n new tokens and lens cached ones (the
    new ones included) of each sequence, `holes` of the table's entries naming
    no page, `pad` rows behind the last sequence."""

    def __init__(self, n, lens, hq, hkv, d, page, dtype, seed=0, pad=0, holes=0.0, first_page=0, spread=1.0):
        self.n, self.lens, self.hq, self.hkv, self.d, self.page, self.dtype = n, lens, hq, hkv, d, page, dtype
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        need = [(l + page - 1) // page for l in lens]
        self.total = first_page + sum(need) + 2
        order = (first_page + r.permutation(sum(need) + 2)).astype(np.uint32)
        width = max(1, max(need)) + 1
        self.table = np.full((len(n), width), NO_PAGE, dtype=np.uint32)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m]
            at += m
        drop = (r.random(self.table.shape) < holes)
        self.table[drop] = r.choice(np.array([NO_PAGE, self.total, 2 ** 31], dtype=np.uint32), drop.sum())
        self.rows = sum(n)
        self.T = max(1, self.rows + pad)
        self.starts = np.concatenate([[0], np.cumsum(n)])
        self.width = width

    def normal(self, *shape, scale=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(self.dtype)

    def batch(self, ops, max_q=None, max_kv=None):
        return ops.PagedBatch(i32(self.table), i32(self.starts), i32(self.lens), self.T,
                              max_q or max(1, max(self.n)), max_kv or max(1, max(self.lens)))

    def rows_of(self):
        """(row, sequence, position) of every token row."""
        for s, (n, l) in enumerate(zip(self.n, self.lens)):
            for i in range(n):
                yield int(self.starts[s]) + i, s, l - n + i


def turned(x, w, pos, eps, theta, rot, halves, inv_freq=None):
    """Norm and rotation of x [heads, D] (float64 in and out)."""
    x = x.double()
    d = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    k = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    ang = pos * (inv_freq if inv_freq is not None else theta ** (-2 * k / max(rot, 1)))
    a, b = ((x[..., :rot // 2], x[..., rot // 2:rot]) if halves else (x[..., 0:rot:2], x[..., 1:rot:2]))
    c, s = ang.cos(), ang.sin()
    u, v = a * c - b * s, a * s + b * c
    y = x.clone()
    if halves:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, v
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    # a bound on what float32 arithmetic and the store may be off: the pair's
    # length times a few float32 steps, half a step of the value, and half the
    # smallest subnormal of f16
    size = torch.zeros_like(x)
    length = torch.sqrt(a * a + b * b)
    size += x.abs()
    if halves:
        size[..., :rot // 2], size[..., rot // 2:rot] = length, length
    else:
        size[..., 0:rot:2], size[..., 1:rot:2] = length, length
    return y, size


def attend(case, k_pages, v_pages, q, row, s, pos, h, scale=0.0, softcap=0.0, window=0, slopes=None, prefix=0):
    """float64 (out [D], lse, weight on |v| [D], keys, size of the scores) of one row and head."""
    hk = h // (case.hq // case.hkv)
    j = np.arange(case.lens[s])
    see = ((j <= pos) | (j < prefix)) & ((j > pos - window) if window else True)
    j = j[see]
    page = case.table[s, j // case.page].astype(np.int64)
    j, page = j[page < case.total], page[page < case.total]
    d = case.d
    if len(j) == 0:
        z = torch.zeros(d, dtype=torch.float64)
        return z, -math.inf, z, 0, 0.0
    at, slot = torch.from_numpy(page).cuda(), torch.from_numpy(j % case.page).cuda()
    k = k_pages[at, hk, slot].double()
    v = v_pages[at, hk, :, slot].double()
    qv = q[row, h].double()
    c = scale or 1 / math.sqrt(d)
    x = (k @ qv) * c
    size = float(((k.abs() @ qv.abs()) * c).max())
    if softcap:
        x = softcap * torch.tanh(x / softcap)
        size += softcap
    if slopes is not None:
        bias = float(slopes[h]) * torch.from_numpy(np.abs(pos - j)).cuda().double()
        x = x - bias
        size += float(bias.max())
    m = x.max()
    if m == -math.inf:
        z = torch.zeros(d, dtype=torch.float64)
        return z, -math.inf, z, len(j), size
    p = torch.exp(x - m)
    l = p.sum()
    return ((p @ v) / l).cpu(), float(m + torch.log(l)), ((p @ v.abs()) / l).cpu(), len(j), size


def attend_tol(case, out, on_v, keys, size, vmax):
    """How far a row's output may be off.  Weights are rounded to the type
    (half a step each, and half of f16's smallest subnormal per key against a
    sum of at least 1); a float32 score is off by at most (D + 8) 2^-24 times
    the sum of its products' sizes, which moves every weight by that factor,
    above and below the line; the store rounds once more."""
    half = HALF_STEP[case.dtype]
    score = (case.d + 8) * 2.0 ** -24 * size + 2.0 ** -21
    return (half + 2 * score) * on_v + keys * 2.0 ** -25 * vmax + half * out.abs() + 2.0 ** -24


def lse_tol(case, lse, keys, size):
    """A float32 score's error (as above) plus the sum's: a lane adds at most
    keys / 16 + 64 weights in a row, then the partial sums."""
    return (case.d + 8) * 2.0 ** -24 * size + (keys / 16 + 100) * 2.0 ** -24 + 2.0 ** -21 * (1 + abs(lse))
