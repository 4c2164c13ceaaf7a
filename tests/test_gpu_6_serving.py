"""GPU parity of the serving operators -- paged append, paged attention, token
log probabilities -- against float64 (tests/serving_ref.py), at the lengths,
masks, strides and page tables where they can go wrong, and of a run of them as
a server uses them."""
import ctypes as C
import itertools
import math
import random

import numpy as np
import pytest
import torch

import serving_ref as R
from nnzap_amd import _lib as L
from nnzap_amd import configs as cf
from nnzap_amd import ops
from nnzap_amd.ops import Device, NnzError

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def same(a, b):
    """Bit for bit, NaN included."""
    view = torch.int16 if a.element_size() == 2 else torch.int32
    return torch.equal(a.contiguous().view(view), b.contiguous().view(view))


# ------------------------------------------------------------------- append
APPENDS = [
    # n, lens, hq, hkv, d, page
    ([1], [701], 16, 8, 128, 16),
    ([1] * 70, [1 + 37 * i for i in range(70)], 4, 2, 64, 16),
    ([5, 0, 33, 1, 16, 0], [5, 0, 40, 1000, 17, 9], 4, 2, 128, 32),
    ([130, 7], [131, 300], 6, 2, 64, 64),
    ([17, 3, 8], [9, 0, 8], 2, 1, 128, 16),           # rows at negative positions
    ([2, 9, 64], [999_999, 131_072, 64], 3, 3, 128, 1024),
    ([0, 0], [3, 0], 2, 2, 64, 16),
]


def _append_case(i, dtype, seed=0, **kw):
    n, lens, hq, hkv, d, page = APPENDS[i]
    c = R.Case(n, lens, hq, hkv, d, page, dtype, seed=seed, pad=3, **kw)
    qkv = c.normal(c.T, (hq + 2 * hkv) * d + 8)
    q = qkv[:, :hq * d].view(c.T, hq, d) if c.T == 1 else qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d].unflatten(1, (hkv, d))
    kp, vp = c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
    return c, q, k, v, kp, vp


def _check_append(c, q, k, v, before, after, q_out, q_before, w, eps, theta, rot, halves, inv_freq=None):
    kp, vp = before[0].double(), before[1].clone()
    tol_k = torch.zeros_like(kp)
    q_ref, tol_q = q_before.double(), torch.zeros(q_before.shape, dtype=torch.float64, device="cuda")
    half = R.HALF_STEP[c.dtype]
    bound = lambda y, size: half * y.abs() + 2.0 ** -20 * size + 2.0 ** -25   # noqa: E731
    for row, s, pos in c.rows_of():
        if pos < 0:
            continue
        y, size = R.turned(q[row], w[0], pos, eps, theta, rot, halves, inv_freq)
        q_ref[row], tol_q[row] = y, bound(y, size)
        page = int(c.table[s, pos // c.page])
        if page >= c.total:
            continue
        y, size = R.turned(k[row], w[1], pos, eps, theta, rot, halves, inv_freq)
        kp[page, :, pos % c.page], tol_k[page, :, pos % c.page] = y, bound(y, size)
        vp[page, :, :, pos % c.page] = v[row]
    assert ((q_out.double() - q_ref).abs() <= tol_q).all()
    assert ((after[0].double() - kp).abs() <= tol_k).all()
    assert same(after[1], vp)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(dev, i, dtype):
    for seed, (norm, halves, rot) in enumerate([(True, False, None), (True, True, None), (False, True, 32),
                                                (True, False, 48), (False, False, 0)]):
        c, q, k, v, kp, vp = _append_case(i, dtype, seed, holes=0.2 if seed == 1 else 0.0)
        w = [1 + 0.3 * torch.randn(c.d, generator=c.g, device="cuda") if norm else None for _ in range(2)]
        kv = ops.PagedKVCache(dev, kp.clone(), vp.clone())
        q_out = c.normal(c.T, c.hq, c.d)
        q_before = q_out.clone()
        r = c.d if rot is None else rot
        ops.dispatch_paged_append(dev, kv, c.batch(ops), q, k, v, q_out, w[0], w[1], eps=1e-5, theta=1e6,
                                  rotary_dim=rot, halves=halves)
        dev.sync()
        _check_append(c, q, k, v, (kp, vp), (kv.k_pages, kv.v_pages), q_out, q_before, w, 1e-5, 1e6, r, halves)


def test_append_in_place_one_scale_and_given_frequencies(dev):
    c, q, k, v, kp, vp = _append_case(2, F16)
    w = [None, torch.rand(c.d, generator=c.g, device="cuda") + 0.5]
    freq = torch.rand(c.d // 2, generator=c.g, device="cuda", dtype=torch.float64) * 2
    kv = ops.PagedKVCache(dev, kp.clone(), vp.clone())
    q_before = q.clone()
    ops.dispatch_paged_append(dev, kv, c.batch(ops), q, k, v, q, w[0], w[1], inv_freq=freq, halves=True)
    dev.sync()
    _check_append(c, q_before, k, v, (kp, vp), (kv.k_pages, kv.v_pages), q, q_before, w, 1e-6, 0.0, c.d, True, freq)


def test_append_follows_the_device_arrays_and_leaves_rows_beyond_the_bounds(dev):
    """One batch object, its arrays changed between calls; a q_len beyond
    max_q_len computes the first max_q_len rows only, a kv_len beyond
    max_kv_len counts as it."""
    c, q, k, v, kp, vp = _append_case(2, F16)
    b = c.batch(ops, max_q=8, max_kv=40)
    kv = ops.PagedKVCache(dev, kp.clone(), vp.clone())
    q_out = torch.zeros_like(q)
    ops.dispatch_paged_append(dev, kv, b, q, k, v, q_out)
    dev.sync()
    done = q_out.abs().amax((1, 2)) > 0
    want = torch.zeros(c.T, dtype=torch.bool)
    for s, (n, st) in enumerate(zip(c.n, c.starts)):
        want[st:st + min(n, 8)] = True
    assert torch.equal(done.cpu(), want)
    b.kv_lens.zero_()
    q_out.zero_()
    ops.dispatch_paged_append(dev, kv, b, q, k, v, q_out)
    dev.sync()
    assert not q_out.any()      # every row is at a negative position


def test_append_agrees_with_the_single_token_operators(dev):
    """A decode step's append equals dispatch_fused_norm_rope and
    dispatch_fused_k_norm_rope_kv_cache to one f16 step of the rotated pair
    (their angles are float32 products)."""
    c = R.Case([1], [301], 16, 8, 128, 16, F16, seed=3)
    q, k, v = c.normal(1, 16, 128), c.normal(1, 8, 128), c.normal(1, 8, 128)
    w = [1 + 0.1 * torch.randn(128, generator=c.g, device="cuda") for _ in range(2)]
    kv = ops.PagedKVCache.empty(dev, c.total, 16, 8, 128)
    q_out = torch.empty_like(q)
    ops.dispatch_paged_append(dev, kv, c.batch(ops), q, k, v, q_out, w[0], w[1], eps=1e-6, theta=1e6)
    kc, vc = torch.zeros(8, 304, 128, dtype=F16, device="cuda"), torch.zeros(8, 128, 304, dtype=F16, device="cuda")
    q1 = q.clone()
    ops.dispatch_fused_norm_rope(dev, q1, w[0], L.FusedNormRoPEDims(16, 128, 300, 1e-6, 1e6))
    ops.dispatch_fused_k_norm_rope_kv_cache(dev, k, v, kc, vc, w[1], L.FusedKNormRoPEKVDims(8, 128, 300, 304, 1e-6, 1e6))
    dev.sync()
    page, slot = int(c.table[0, 300 // 16]), 300 % 16
    # angle error of the float32 operators: 300 * 2^-24 radians of a pair of at most ~5
    for a, b in ((q_out, q1), (kv.k_pages[page, :, slot], kc[:, 300])):
        assert ((a.double() - b.double()).abs() <= 2.0 ** -10 * b.double().abs() + 1e-3).all()
    assert same(kv.v_pages[page, :, :, slot], vc[:, :, 300])


# ---------------------------------------------------------------- attention
ATTENTION = {
    # name: n, lens, hq, hkv, d, page
    "one": ([1], [1], 2, 2, 64, 16),
    "one_513": ([1], [513], 16, 8, 128, 16),
    "decode": ([1] * 9, [3, 16, 17, 250, 1000, 31, 32, 33, 4100], 8, 2, 128, 16),
    "decode_64": ([1] * 5, [700, 64, 2, 129, 1023], 4, 4, 64, 32),
    "decode_odd_group": ([1, 0, 1], [300, 40, 77], 6, 2, 128, 64),
    "decode_wide_group": ([1, 1], [300, 2100], 40, 2, 64, 128),
    "drafts": ([4, 2, 3, 4], [4, 130, 67, 900], 8, 2, 128, 16),
    "drafts_over_16_rows": ([5, 4, 1, 5], [37, 130, 667, 5], 8, 2, 64, 16),
    "prompt": ([65], [65], 4, 2, 128, 16),
    "prompts": ([130, 1, 200, 0, 63], [130, 1, 200, 0, 64], 4, 1, 64, 64),
    "chunk": ([150], [1150], 8, 8, 128, 16),
    "mixed": ([1, 97, 1, 40, 3], [700, 1200, 1, 40, 2000], 8, 2, 128, 32),
    "short_of_keys": ([6, 30], [2, 7], 4, 2, 64, 16),      # the first rows see nothing
}
OPTIONS = [dict(), dict(softcap=12.0), dict(window=50), dict(bias=True), dict(prefix=40),
           dict(softcap=30.0, window=7, bias=True, prefix=90, scale=0.3), dict(holes=0.3), dict(window=1)]


def _attention(dev, c, kp, vp, q, ws=None, lse=True, **o):
    kv, b = ops.PagedKVCache(dev, kp, vp), c.batch(ops)
    out = torch.full((c.T, c.hq, c.d), 7.0, dtype=c.dtype, device="cuda")
    ls = torch.full((c.T, c.hq), 7.0, device="cuda") if lse else None
    if ws is None:
        n = ops.paged_attention_workspace_bytes(kv, b, c.hq)
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")   # NaN throughout
    ops.dispatch_paged_attention(dev, kv, b, q, out, ws, lse=ls, **o)
    dev.sync()
    return out, ls


def _check_attention(c, kp, vp, q, out, lse, rows=None, **o):
    prefix = o.pop("prefix_lens", None)
    vmax = float(torch.nan_to_num(vp.double(), 0, 0, 0).abs().max())
    picked = list(c.rows_of())
    if rows:
        picked = random.Random(5).sample(picked, min(rows, len(picked)))
        picked += [list(c.rows_of())[-1]]
    for row, s, pos in picked:
        for h in {0, c.hq - 1, row % c.hq}:
            want, want_lse, on_v, keys, size = R.attend(
                c, kp, vp, q, row, s, pos, h, prefix=int(prefix[s]) if prefix is not None else 0, **o)
            got = out[row, h].double().cpu()
            tol = R.attend_tol(c, want, on_v, keys, size, vmax) if keys else torch.zeros(c.d)
            assert ((got - want).abs() <= tol).all(), (row, s, pos, h, float((got - want).abs().max()))
            if lse is not None:
                if want_lse == -math.inf:
                    assert float(lse[row, h]) == -math.inf
                else:
                    assert abs(float(lse[row, h]) - want_lse) <= R.lse_tol(c, want_lse, keys, size)
    assert (out[c.rows:] == 7.0).all()
    assert lse is None or (lse[c.rows:] == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", ATTENTION)
def test_attention(dev, name, dtype):
    n, lens, hq, hkv, d, page = ATTENTION[name]
    for seed, o in enumerate(OPTIONS):
        o = dict(o)
        print(f"attention {name} {dtype} {o}", flush=True)
        c = R.Case(n, lens, hq, hkv, d, page, dtype, seed=seed, pad=2, holes=o.pop("holes", 0.0))
        if o.pop("bias", False):
            o["slopes"] = torch.rand(hq, generator=c.g, device="cuda") * 0.2
        if "prefix" in o:
            first = o.pop("prefix")
            o["prefix_lens"] = torch.tensor([first + 3 * s for s in range(len(n))], dtype=torch.int32, device="cuda")
        q = c.normal(c.T, hq * d + 24)[:, :hq * d].unflatten(1, (hq, d))
        kp, vp = c.normal(c.total, hkv, page, d, scale=1.5), c.normal(c.total, hkv, d, page)
        out, lse = _attention(dev, c, kp, vp, q, **o)
        _check_attention(c, kp, vp, q, out, lse, rows=24, **o)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", ["decode", "drafts", "drafts_over_16_rows", "prompts", "mixed"])
def test_what_masked_positions_hold_has_no_influence(dev, name, dtype):
    """NaN and infinities in every slot behind a sequence's end, in unused
    pages and before its window, in K and in V; then in a key that later rows
    of a chunk see and earlier ones do not."""
    n, lens, hq, hkv, d, page = ATTENTION[name]
    c = R.Case(n, lens, hq, hkv, d, page, dtype, seed=4)
    q = c.normal(c.T, hq, d)
    kp, vp = c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
    clean, clean_lse = _attention(dev, c, kp, vp, q, window=40)
    seen = torch.zeros(c.total, page, dtype=torch.bool)
    for row, s, pos in c.rows_of():
        for j in range(max(0, pos - 39), pos + 1):
            seen[int(c.table[s, j // page]), j % page] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=dtype)
    dirt = bad[torch.randint(0, 3, (c.total, hkv, page, d), generator=c.g, device="cuda")]
    hidden = ~seen.cuda()[:, None, :, None]
    kd = torch.where(hidden, dirt, kp).contiguous()
    vd = torch.where(hidden.transpose(2, 3), dirt.transpose(2, 3), vp).contiguous()
    out, lse = _attention(dev, c, kd, vd, q, window=40)
    assert same(out, clean) and same(lse, clean_lse)
    for row, s, pos in list(c.rows_of()):
        if pos == lens[s] - 1 and n[s] > 1:
            vp = vp.clone()
            page_, slot = int(c.table[s, pos // page]), pos % page
            vp[page_, :, 0, slot], vp[page_, :, 1, slot], vp[page_, :, 2, slot] = math.nan, math.inf, -math.inf
    out2, lse2 = _attention(dev, c, kp, vp, q, window=40)
    assert same(lse2, clean_lse)
    for row, s, pos in c.rows_of():
        if pos == lens[s] - 1 and n[s] > 1:
            assert out2[row, :, 0].isnan().all()
            assert (out2[row, :, 1] == math.inf).all() and (out2[row, :, 2] == -math.inf).all()
            assert same(out2[row, :, 3:], clean[row, :, 3:])
        else:
            assert same(out2[row], clean[row])


@pytest.mark.parametrize("name", ["decode", "mixed"])
def test_infinite_and_nan_scores(dev, name):
    """A visible NaN key makes its rows NaN; keys whose scores are all -inf make
    a row of zeros with lse -inf, and such a key among others is ignored."""
    n, lens, hq, hkv, d, page = ATTENTION[name]
    c = R.Case(n, lens, hq, hkv, d, page, F16, seed=6)
    q = c.normal(c.T, hq, d).abs() + 0.1
    kp, vp = c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
    page0 = [int(c.table[s, 0]) for s in range(len(n))]
    k1 = kp.clone()
    k1[page0, :, 0] = -math.inf
    out, lse = _attention(dev, c, k1, vp, q)
    k2 = kp.clone()
    k2[page0, :, 0] = math.nan
    nan_out, nan_lse = _attention(dev, c, k2, vp, q)
    assert nan_out[:c.rows].isnan().all() and nan_lse[:c.rows].isnan().all()
    for row, s, pos in c.rows_of():
        if pos == 0:
            assert not out[row].any() and (lse[row] == -math.inf).all()
    _check_attention(c, k1, vp, q, out, lse, rows=12)
    all_low = torch.full_like(kp, -math.inf)
    out, lse = _attention(dev, c, all_low, vp, q)
    assert not out[:c.rows].any() and (lse[:c.rows] == -math.inf).all()


def test_large_scores(dev):
    """Scores of several hundred that climb and fall along the keys: the running
    maximum moves at every step, or far below it nothing is left."""
    for dtype, d in ((F16, 128), (BF16, 64)):
        c = R.Case([1, 70, 3], [3000, 600, 513], 4, 2, d, 16, dtype, seed=8)
        q = c.normal(c.T, 4, d)
        kp, vp = c.normal(c.total, 2, 16, d, scale=30.0), c.normal(c.total, 2, d, 16)
        for s in range(3):
            for e in range(c.lens[s] // 16):
                kp[int(c.table[s, e])] *= 0.05 + e / 60.0 if s != 1 else 2.0 - e / 30.0
        out, lse = _attention(dev, c, kp, vp, q)
        _check_attention(c, kp, vp, q, out, lse, rows=20)


def test_attention_stays_within_the_hosts_bounds(dev):
    """Arrays on the device that pass the bounds of the host: of a longer q_len
    the first max_q_len rows are computed, at the positions that the arrays say;
    a longer kv_len counts as max_kv_len; other rows keep what they hold."""
    for name, max_q in (("mixed", 20), ("drafts", 2), ("prompts", 64)):
        n, lens, hq, hkv, d, page = ATTENTION[name]
        c = R.Case(n, lens, hq, hkv, d, page, F16, seed=12, pad=2)
        q, kp, vp = c.normal(c.T, hq, d), c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
        want, _ = _attention(dev, c, kp, vp, q)
        kv, b = ops.PagedKVCache(dev, kp, vp), c.batch(ops, max_q=max_q)
        out = torch.full((c.T, hq, d), 7.0, dtype=F16, device="cuda")
        ws = torch.full((max(16, ops.paged_attention_workspace_bytes(kv, b, hq)),), 255, dtype=torch.uint8, device="cuda")
        ops.dispatch_paged_attention(dev, kv, b, q, out, ws)
        dev.sync()
        for s, (m, st) in enumerate(zip(n, c.starts)):
            _near(out[st:st + min(m, max_q)], want[st:st + min(m, max_q)])
            assert (out[st + min(m, max_q):st + m] == 7.0).all()
        assert (out[c.rows:] == 7.0).all()
        short = max(1, max(lens) // 2)
        b = c.batch(ops, max_kv=short)
        d2 = R.Case(n, [min(l, short) for l in lens], hq, hkv, d, page, F16, seed=12, pad=2)
        d2.table, d2.total = c.table, c.total
        out = torch.full((c.T, hq, d), 7.0, dtype=F16, device="cuda")
        lse = torch.full((c.T, hq), 7.0, device="cuda")
        ops.dispatch_paged_attention(dev, kv, b, q, out, ws.new_full((max(16, ops.paged_attention_workspace_bytes(kv, b, hq)),), 255), lse=lse)
        dev.sync()
        _check_attention(d2, kp, vp, q, out, lse, rows=16)


def _near(a, b):
    """Two calls that split the same keys differently: their float32 sums differ by
    the order, and by what weights and stores then round to (half a step each way)."""
    assert ((a.double() - b.double()).abs() <= 4 * 2.0 ** -11 * b.double().abs().amax(-1, keepdim=True) + 1e-6).all()


@pytest.mark.parametrize("page", [256, 1024])
def test_attention_over_large_pages_into_strided_rows(dev, page):
    c = R.Case([1, 70, 2], [2100, 500, 1030], 6, 2, 64, page, BF16, seed=13)
    q, kp, vp = c.normal(c.T, 6, 64), c.normal(c.total, 2, page, 64), c.normal(c.total, 2, 64, page)
    kv, b = ops.PagedKVCache(dev, kp, vp), c.batch(ops)
    rows = torch.full((c.T, 6 * 64 + 40), 7.0, dtype=BF16, device="cuda")
    out = rows[:, 8:8 + 6 * 64].unflatten(1, (6, 64))
    lse = torch.zeros(c.T, 6, device="cuda")
    ws = torch.full((max(16, ops.paged_attention_workspace_bytes(kv, b, 6)),), 255, dtype=torch.uint8, device="cuda")
    ops.dispatch_paged_attention(dev, kv, b, q, out, ws, lse=lse)
    dev.sync()
    _check_attention(c, kp, vp, q, out, lse, rows=16)
    assert (rows[:, :8] == 7.0).all() and (rows[:, 8 + 6 * 64:] == 7.0).all()


def test_many_sequences(dev):
    """More sequences than a wave looks through at once, some of them empty."""
    r = random.Random(3)
    n = [r.choice([0, 0, 1, 1, 2, 17]) for _ in range(300)]
    lens = [m + r.randint(0, 60) for m in n]
    c = R.Case(n, lens, 4, 2, 64, 16, F16, seed=14, pad=5)
    q, kp, vp = c.normal(c.T, 4, 64), c.normal(c.total, 2, 16, 64), c.normal(c.total, 2, 64, 16)
    out, lse = _attention(dev, c, kp, vp, q)
    _check_attention(c, kp, vp, q, out, lse, rows=40)
    k, v = c.normal(c.T, 2, 64), c.normal(c.T, 2, 64)
    kv = ops.PagedKVCache(dev, kp.clone(), vp.clone())
    q_out = torch.zeros_like(q)
    ops.dispatch_paged_append(dev, kv, c.batch(ops), q, k, v, q_out, rotary_dim=0)
    dev.sync()
    ks, vs = kp.clone(), vp.clone()
    for row, s, pos in c.rows_of():
        p = int(c.table[s, pos // 16])
        ks[p, :, pos % 16], vs[p, :, :, pos % 16] = k[row], v[row]
    assert same(kv.k_pages, ks) and same(kv.v_pages, vs)
    assert same(q_out[:c.rows], q[:c.rows]) and not q_out[c.rows:].any()


def test_far_pages(dev):
    """Pages whose byte offsets pass 32 bits, in K and in V."""
    c = R.Case([1, 90], [900, 300], 8, 8, 128, 16, F16, seed=2, first_page=140_000)
    kp = torch.zeros(c.total, 8, 16, 128, dtype=F16, device="cuda")
    vp = torch.zeros(c.total, 8, 128, 16, dtype=F16, device="cuda")
    kp[140_000:], vp[140_000:] = c.normal(c.total - 140_000, 8, 16, 128), c.normal(c.total - 140_000, 8, 128, 16)
    assert 140_000 * 8 * 16 * 128 * 2 > 2 ** 32
    q = c.normal(c.T, 8, 128)
    out, lse = _attention(dev, c, kp, vp, q)
    _check_attention(c, kp, vp, q, out, lse, rows=20)
    k, v = c.normal(c.T, 8, 128), c.normal(c.T, 8, 128)
    kv = ops.PagedKVCache(dev, kp, vp)
    ops.dispatch_paged_append(dev, kv, c.batch(ops), q, k, v, out, rotary_dim=0)
    dev.sync()
    for row, s, pos in c.rows_of():
        page = int(c.table[s, pos // 16])
        assert same(kp[page, :, pos % 16], k[row]) and same(vp[page, :, :, pos % 16], v[row])
    assert same(out, q)


def test_long_context_splits(dev):
    """One and two sequences over long caches: the split over keys and its join."""
    for dtype, n, lens, o in ((F16, [1], [70_001], {}), (BF16, [3, 1], [33_000, 90], dict(softcap=20.0)),
                              (F16, [40], [20_011], {}), (F16, [1, 20], [30_000, 9000], dict(window=5000))):
        c = R.Case(n, lens, 8, 2, 128, 64, dtype, seed=9)
        q = c.normal(c.T, 8, 128)
        kp, vp = c.normal(c.total, 2, 64, 128), c.normal(c.total, 2, 128, 64)
        out, lse = _attention(dev, c, kp, vp, q, **o)
        _check_attention(c, kp, vp, q, out, lse, rows=4, **o)


@pytest.mark.parametrize("d,hq,hkv,n,lens", [
    (64, 2, 2, [1], [6001]), (128, 4, 4, [16], [5999]), (128, 2, 2, [300], [6050]), (64, 4, 2, [129], [6127]),
    (64, 2, 2, [1, 200, 16], [6100, 3333, 6031])])
def test_windows_wherever_they_begin(dev, d, hq, hkv, n, lens):
    """Keys are split by what a window can show; rows whose keys begin and end
    anywhere in the steps and tiles of that see all of them."""
    for shift, window in enumerate((1, 481, 512, 513, 1023, 2000, 2017, 5000, 2**32 - 1)):
        c = R.Case(n, [x - 13 * shift for x in lens], hq, hkv, d, 32, F16, seed=shift)
        q = c.normal(c.T, hq, d)
        kp, vp = c.normal(c.total, hkv, 32, d), c.normal(c.total, hkv, d, 32)
        out, lse = _attention(dev, c, kp, vp, q, window=window)
        _check_attention(c, kp, vp, q, out, lse, rows=6, window=window)


def test_attention_agrees_with_the_contiguous_operator(dev):
    """A decode step over pages equals nnz_dispatch_gqa_attention on the same
    tokens in one contiguous cache, to the rounding of weights and store."""
    q_, k_, v_ = cf.config4(704)
    bf = lambda a: torch.from_numpy(a.view(np.int16)).cuda().view(BF16)   # noqa: E731
    q, k, v = bf(q_), bf(k_), bf(v_)
    dims = L.GQADims(16, 8, 128, 704, 704, 2)
    ref = torch.empty(16, 128, device="cuda")
    scratch = torch.empty((ops.gqa_scratch_bytes(dims) + 3) // 4, device="cuda")
    ops.dispatch_gqa_attention(dev, q, k, v, ref, scratch, dims, v_transposed=False)
    c = R.Case([1], [704], 16, 8, 128, 16, BF16, seed=1)
    kp = torch.zeros(c.total, 8, 16, 128, dtype=BF16, device="cuda")
    vp = torch.zeros(c.total, 8, 128, 16, dtype=BF16, device="cuda")
    for j in range(704):
        page = int(c.table[0, j // 16])
        kp[page, :, j % 16], vp[page, :, :, j % 16] = k[:, j], v[:, j]
    out, _ = _attention(dev, c, kp, vp, q[None])
    _check_attention(c, kp, vp, q[None], out, None)
    # both against the same float64: their difference is within twice the weights' and the store's half step
    assert ((out[0].double() - ref.double()).abs() <= 2 * 2.0 ** -8 * (ref.double().abs() + float(v.abs().max()))).all()


def test_attention_refuses_a_short_workspace(dev):
    c = R.Case([1], [70_001], 8, 2, 128, 64, F16)
    q = c.normal(c.T, 8, 128)
    kv = ops.PagedKVCache(dev, c.normal(c.total, 2, 64, 128), c.normal(c.total, 2, 128, 64))
    n = ops.paged_attention_workspace_bytes(kv, c.batch(ops), 8)
    assert n > 0
    for ws in (None, torch.zeros(n - 1, dtype=torch.uint8, device="cuda"),
               torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[8:]):
        with pytest.raises(NnzError, match="workspace"):
            ops.dispatch_paged_attention(dev, kv, c.batch(ops), q, torch.empty_like(q), ws)


def test_calls_repeat_bit_for_bit(dev):
    for name in ("decode", "mixed"):
        n, lens, hq, hkv, d, page = ATTENTION[name]
        c = R.Case(n, lens, hq, hkv, d, page, F16, seed=5)
        q, kp, vp = c.normal(c.T, hq, d), c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
        a, la = _attention(dev, c, kp, vp, q)
        for _ in range(3):
            b, lb = _attention(dev, c, kp, vp, q)
            assert same(a, b) and same(la, lb)


# --------------------------------------------------------------- logprobs
def _logprobs(dev, x, tok, top, T=1.0):
    rows, vocab = x.shape
    f = lambda *s: torch.full(s, 7.0, device="cuda")   # noqa: E731
    i = lambda *s: torch.full(s, 7, dtype=torch.int32, device="cuda")   # noqa: E731
    o = dict(lse=f(rows), entropy=f(rows), rank=i(rows))
    if top:
        o.update(top_ids=i(rows, top), top_logprobs=f(rows, top))
    lp = f(rows)
    ws = torch.full((max(16, ops.token_logprobs_workspace_bytes(rows, vocab, top)),), 255, dtype=torch.uint8,
                    device="cuda")
    ops.dispatch_token_logprobs(dev, x, tok, lp, ws, temperature=T, **o)
    dev.sync()
    return dict(lp=lp, **o)


def _check_logprobs(x, tok, got, top, T=1.0):
    """float64 on the host.  A float32 sum over a lane's vocab / 64 values, then
    of the lanes, is off by at most vocab / 64 half steps of 2^-24; a value
    (x - max) / T by two steps of its size, and entropy weighs such values."""
    vocab = x.shape[1]
    sums = (vocab / 64 + 64) * 2.0 ** -24
    for r, row in enumerate(x.double().cpu().numpy()):
        t = int(np.uint32(tok[r].item() & 0xFFFFFFFF))
        poisoned = np.isnan(row).any() or (row == math.inf).any()
        none = not poisoned and (row == -math.inf).all()
        keep = np.flatnonzero(~np.isnan(row))
        order = keep[np.lexsort((keep, -row[keep]))]
        full = np.concatenate([order, np.flatnonzero(np.isnan(row))])
        rank = int(np.flatnonzero(full == t)[0]) if t < vocab else vocab
        assert int(got["rank"][r]) == rank, (r, t)
        m = row.max() if not poisoned else 0.0
        if none:
            lse, lp, H = -math.inf, np.full(vocab, -math.inf), 0.0
        elif not poisoned:
            y = (row - m) / T
            lse = m / T + math.log(np.exp(y).sum())
            lp = y - math.log(np.exp(y).sum())
            with np.errstate(invalid="ignore"):
                H = float(-np.where(np.exp(lp) > 0, np.exp(lp) * lp, 0).sum())

        def near(a, b):
            if poisoned:
                return math.isnan(a)
            if math.isinf(b):
                return a == b
            return abs(a - b) <= sums + 2.0 ** -21 * (1 + abs(b) + abs(m / T))
        assert near(float(got["lp"][r]), lp[t] if t < vocab and not poisoned else -math.inf), (r, t)
        assert near(float(got["lse"][r]), lse if not poisoned else 0)
        if poisoned:
            assert math.isnan(float(got["entropy"][r]))
        else:
            spread = float((np.exp(lp[lp > -700]) * np.abs(y[lp > -700])).sum()) if not none else 0.0
            assert abs(float(got["entropy"][r]) - H) <= 2 * sums * (1 + spread) + 2.0 ** -20 * (1 + spread)
        if top:
            ids = got["top_ids"][r].cpu().numpy().view(np.uint32)
            want = np.full(top, 0xFFFFFFFF, dtype=np.uint32)
            want[:min(top, len(order))] = order[:top]
            assert np.array_equal(ids, want), (r, ids, want)
            for j, i in enumerate(want):
                v = float(got["top_logprobs"][r, j])
                assert math.isnan(v) if i == 0xFFFFFFFF else near(v, lp[i] if not poisoned else 0.0)


SIZES = [(1, 1), (3, 2), (2, 5), (4, 63), (3, 64), (5, 65), (2, 255), (7, 1000), (3, 4097), (2, 50257), (1, 151669),
         (90, 3001), (300, 17_001)]


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_logprobs(dev, rows, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for k, (top, pad, T) in enumerate([(0, 0, 1.0), (1, 1, 0.7), (min(5, vocab), 3, 1.3), (min(64, vocab), 8, 1.0)]):
        print(f"logprobs {rows} x {vocab} {dtype} top {top}", flush=True)
        buf = (torch.randn(rows, vocab + pad, generator=g, device="cuda") * 4).to(dtype)
        x = buf[:, pad:] if k % 2 else buf[:, :vocab]
        tok = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        _check_logprobs(x, tok, _logprobs(dev, x, tok, top, T), top, T)


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
def test_logprobs_of_masked_tied_and_poisoned_rows(dev, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    for vocab in (70, 4999):
        x = (torch.randn(16, vocab, generator=g, device="cuda") * 3).to(dtype)
        low = torch.finfo(dtype).min
        x[0] = -math.inf                           # nothing left
        x[1] = low                                 # masked throughout by the lowest value
        x[2] = 1.5                                 # all tied
        x[3, ::2] = -math.inf
        x[4, 1:] = low                             # one left
        x[5, 1:] = -math.inf
        x[6] = x[6].round()                        # many ties
        x[7, 11] = math.nan
        x[8, 12] = math.inf
        x[9] = math.nan
        x[10, 3:] = math.nan
        x[11, 20] = -math.inf
        x[12] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, 0.0, -0.0).to(dtype)
        x[13] = torch.arange(vocab, device="cuda").to(dtype) / 64      # rising: every element enters the list
        x[14] = -torch.arange(vocab, device="cuda").to(dtype) / 64
        tok = torch.randint(0, vocab, (16,), generator=g, device="cuda", dtype=torch.int32)
        for t in (tok, torch.full_like(tok, vocab - 1), torch.zeros_like(tok), torch.full_like(tok, 20),
                  torch.full_like(tok, vocab), torch.full_like(tok, -1)):
            for top in (0, 7, 64):
                _check_logprobs(x, t, _logprobs(dev, x, t, top), top)


def test_logprobs_of_far_rows(dev):
    """Rows whose byte offsets pass 32 bits."""
    stride = 151_936
    buf = torch.empty(7200, stride, device="cuda")
    buf[:4].normal_()
    buf[-4:].normal_()
    for rows in (slice(0, 4), slice(7196, 7200)):
        want = _logprobs(dev, buf[rows].clone(), torch.arange(4, device="cuda", dtype=torch.int32), 3)
        x = torch.as_strided(buf, (2, stride), (stride * 7196, 1)) if rows.start == 0 else None
        if x is not None:
            got = _logprobs(dev, x, torch.tensor([0, 0], device="cuda", dtype=torch.int32), 3)
            far = _logprobs(dev, buf[7196:7197].clone(), torch.zeros(1, device="cuda", dtype=torch.int32), 3)
            assert torch.equal(got["top_ids"][0], want["top_ids"][0])
            assert torch.equal(got["top_ids"][1], far["top_ids"][0])
            assert abs(float(got["lp"][1]) - float(far["lp"][0])) <= 1e-4


def test_logprobs_refuses_a_short_workspace(dev):
    x, tok = torch.randn(300, 20_000, device="cuda"), torch.zeros(300, dtype=torch.int32, device="cuda")
    n = ops.token_logprobs_workspace_bytes(300, 20_000, 20)
    assert n > 0
    ids = torch.zeros(300, 20, dtype=torch.int32, device="cuda")
    for ws in (None, torch.zeros(n - 1, dtype=torch.uint8, device="cuda"),
               torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[8:]):
        with pytest.raises(NnzError, match="workspace"):
            ops.dispatch_token_logprobs(dev, x, tok, torch.zeros(300, device="cuda"), ws, top_ids=ids)


# ------------------------------------------------- used together, as a server does
class Layer:
    """One attention layer and a 1-bit LM head over paged caches."""

    def __init__(self, dev, dtype=F16, hq=8, hkv=2, d=128, page=16, pages=64, vocab=640, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dev, self.hq, self.hkv, self.d, self.dtype, self.vocab = dev, hq, hkv, d, dtype, vocab
        H = hq * d
        self.w = torch.randn(H, (hq + 2 * hkv) * d, generator=g, device="cuda") / math.sqrt(H)
        self.qn, self.kn = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
        self.head = ops.DeviceQWeight(dev, cf.q1_matrix(vocab, H, 128, 3, 4))
        self.kv = ops.PagedKVCache.empty(dev, pages, page, hkv, d, dtype)

    def step(self, x, batch, ws, stream_sync=False):
        """x f32 [rows, H] -> (attention output, logits f32 [rows, vocab])."""
        T, d = x.shape[0], self.d
        qkv = (x @ self.w).to(self.dtype)
        a, b = self.hq * d, (self.hq + self.hkv) * d
        q, k, v = (t.unflatten(1, (-1, d)) for t in (qkv[:, :a], qkv[:, a:b], qkv[:, b:]))
        out = torch.zeros(T, self.hq, d, dtype=self.dtype, device="cuda")
        ops.dispatch_paged_append(self.dev, self.kv, batch, q, k, v, q, self.qn, self.kn)
        ops.dispatch_paged_attention(self.dev, self.kv, batch, q, out, ws)
        logits = torch.zeros(T, self.vocab, device="cuda")
        ops.dispatch_dequant_gemm(self.dev, self.head, out.view(T, -1).half(), logits, L.GEMM_STORE_F32)
        return out, logits


def test_chunks_and_single_tokens_give_what_whole_prompts_give(dev):
    """Three sequences of one layer: whole prompts in one call; then, in a cache
    with other pages, in ragged chunks and at last token by token.  Outputs,
    logits and log probabilities agree."""
    m, m2 = Layer(dev), Layer(dev)
    lens = [150, 37, 64]
    g = torch.Generator(device="cuda").manual_seed(7)
    xs = [torch.randn(l, 1024, generator=g, device="cuda") for l in lens]
    need = [(l + 15) // 16 for l in lens]

    def table(order):
        t, at = np.full((3, 12), R.NO_PAGE, dtype=np.uint32), 0
        for s in range(3):
            t[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
        return t

    def run(layer, tab, cuts):
        done, outs, logits = [0, 0, 0], [[], [], []], [[], [], []]
        for cut in cuts:
            n = [min(c, l - d) for c, l, d in zip(cut, lens, done)]
            rows = torch.cat([x[d:d + c] for x, d, c in zip(xs, done, n)])
            pad = torch.zeros((-len(rows)) % 4 + 1, 1024, device="cuda")
            rows = torch.cat([rows, pad])
            done = [d + c for d, c in zip(done, n)]
            b = ops.PagedBatch(R.i32(tab), R.i32(np.concatenate([[0], np.cumsum(n)])), R.i32(done), len(rows),
                               max(n), max(done))
            ws = torch.full((max(16, ops.paged_attention_workspace_bytes(layer.kv, b, 8)),), 255, dtype=torch.uint8,
                            device="cuda")
            o, lg = layer.step(rows, b, ws)
            at = 0
            for s in range(3):
                outs[s].append(o[at:at + n[s]])
                logits[s].append(lg[at:at + n[s]])
                at += n[s]
        dev.sync()
        return torch.cat([torch.cat(o) for o in outs]), torch.cat([torch.cat(x) for x in logits])

    r = np.random.default_rng(3)
    whole, lw = run(m, table(r.permutation(64).astype(np.uint32)), [(150, 37, 64)])
    parts, lp = run(m2, table(r.permutation(64).astype(np.uint32)),
                    [(70, 5, 0), (60, 20, 33), (3, 4, 2)] + [(1, 1, 1)] * 29)
    # the two differ by the order of float32 sums, and by what weights and
    # stores then round to: two half steps of the values' size each
    size = whole.double().abs().max(-1, keepdim=True).values
    assert ((whole.double() - parts.double()).abs() <= 4 * 2.0 ** -11 * size + 2.0 ** -11 * 4).all()
    tok = lw.argmax(1).to(torch.int32)
    a, b = _logprobs(dev, lw, tok, 5), _logprobs(dev, lp, tok, 5)
    _check_logprobs(lw, tok, a, 5)
    # a logit sums 1024 outputs that are each off by at most 2^-9 of their size, times scales up to 0.05
    spread = 2.0 ** -9 * 0.05 * whole.double().abs().flatten(1).sum(1)
    assert ((a["lp"] - b["lp"]).double().abs() <= 2 * spread + 1e-4).all()
    assert (a["rank"] == 0).all()


def test_captured_steps_follow_the_lengths_on_the_device():
    """A decode step captured once (append, attention, log probabilities) and
    replayed while the lengths on the device grow equals the eager calls; two
    graphs with a workspace each are replayed in turn with eager work between."""
    dev = Device(0)
    m, e = Layer(dev, pages=200, vocab=640), Layer(dev, pages=200, vocab=640)
    g = torch.Generator(device="cuda").manual_seed(1)
    tab = np.random.default_rng(2).permutation(200)[:3 * 60].astype(np.uint32).reshape(3, 60)
    lens = np.array([500, 17, 300])
    kv0 = torch.randn(200, 2, 16, 128, generator=g, device="cuda").half()
    for x in (m, e):
        x.kv.k_pages.copy_(kv0)
        x.kv.v_pages.copy_(kv0.transpose(2, 3))
    d, T = 128, 3

    class Graph:
        def __init__(self):
            self.batch = ops.PagedBatch(R.i32(tab), R.i32([0, 1, 2, 3]), R.i32(lens), T, 1, 900)
            self.ws = torch.full((max(16, ops.paged_attention_workspace_bytes(m.kv, self.batch, 8)),), 255,
                                 dtype=torch.uint8, device="cuda")
            n = ops.token_logprobs_workspace_bytes(T, 640, 5)
            self.ws2 = torch.full((max(16, n),), 255, dtype=torch.uint8, device="cuda")
            z = lambda *s, t=F16: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
            self.q, self.k, self.v, self.out = z(T, 8, d), z(T, 2, d), z(T, 2, d), z(T, 8, d)
            self.logits, self.lp = z(T, 640, t=torch.float32), z(T, t=torch.float32)
            self.tok, self.ids = z(T, t=torch.int32), z(T, 5, t=torch.int32)
            torch.cuda.synchronize()
            dev.call("nnz_graph_begin")
            self.calls(m, self.ws, self.ws2)
            h = C.c_void_p()
            dev.call("nnz_graph_end", C.byref(h))
            self.h = h

        def calls(self, layer, ws, ws2):
            ops.dispatch_paged_append(dev, layer.kv, self.batch, self.q, self.k, self.v, self.out, layer.qn, layer.kn)
            # the append's output is the attention's query: a buffer of its own
            ops.dispatch_paged_attention(dev, layer.kv, self.batch, self.out, self.q, ws)
            ops.dispatch_dequant_gemm(dev, layer.head, self.q.view(T, -1), self.logits, L.GEMM_STORE_F32)
            ops.dispatch_token_logprobs(dev, self.logits, self.tok, self.lp, ws2, top_ids=self.ids)

        def load(self, x):
            self.q.copy_(x[:, :1024].view(T, 8, d))
            self.k.copy_(x[:, 1024:1280].view(T, 2, d))
            self.v.copy_(x[:, 1280:].view(T, 2, d))
            self.tok.fill_(3)

    a, b = Graph(), Graph()
    eager_ws = torch.full_like(a.ws, 255)
    eager_ws2 = torch.full_like(a.ws2, 255)
    for step in range(8):
        now = lens + 40 * step
        gr = (a, b)[step % 2]
        x = torch.randn(T, 1536, generator=g, device="cuda").half()
        gr.batch.kv_lens.copy_(R.i32(now))
        gr.load(x)
        dev.call("nnz_graph_replay", gr.h)
        dev.sync()
        got = [t.clone() for t in (gr.q, gr.logits, gr.lp, gr.ids)]
        gr.load(x)
        gr.calls(e, eager_ws, eager_ws2)
        dev.sync()
        for u, w in zip(got, (gr.q, gr.logits, gr.lp, gr.ids)):
            assert same(u, w), step
        assert same(m.kv.k_pages, e.kv.k_pages) and same(m.kv.v_pages, e.kv.v_pages)
    for gr in (a, b):
        L.lib().nnz_graph_destroy(gr.h)


def test_two_streams_with_a_workspace_each(dev):
    """Two contexts on two streams, calls interleaved without waiting."""
    d2 = Device(0, own_stream=True)
    n, lens, hq, hkv, d, page = ATTENTION["decode"]
    c = R.Case(n, lens, hq, hkv, d, page, F16, seed=11)
    qs = [c.normal(c.T, hq, d) for _ in range(6)]
    kp, vp = c.normal(c.total, hkv, page, d), c.normal(c.total, hkv, d, page)
    want = [_attention(dev, c, kp, vp, q)[0] for q in qs]
    b = c.batch(ops)
    outs = [torch.zeros_like(q) for q in qs]
    kvs = [ops.PagedKVCache(x, kp, vp) for x in (dev, d2)]
    wss = [torch.full((max(16, ops.paged_attention_workspace_bytes(kvs[0], b, hq)),), 255, dtype=torch.uint8,
                      device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for i, (q, o) in enumerate(zip(qs, outs)):
        ops.dispatch_paged_attention((dev, d2)[i % 2], kvs[i % 2], b, q, o, wss[i % 2])
    dev.sync()
    d2.sync()
    assert all(same(o, w) for o, w in zip(outs, want))
    d2.close()
