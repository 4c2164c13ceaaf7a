"""CPU checks of the serving operators: what they refuse, and the index
arithmetic their kernels rely on (nnzap_amd/csrc/paged.h, compiled for the
host), with device arrays that break their promises among the inputs."""
import ctypes as C
import random
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from nnzap_amd import _lib as L
from nnzap_amd import ops
from nnzap_amd.ops import NnzError

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def h(tmp_path_factory):
    so = tmp_path_factory.mktemp("paged") / "paged_host.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                    str(HERE / "c" / "paged_host.cc"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    for f in (lib.h_append, lib.h_attn, lib.h_logprobs):
        f.restype = C.c_int
    return lib


def u32s(*v):
    return (C.c_uint32 * len(v))(*v)


A = 0x1000   # an aligned address that is never followed


def kv(**c):
    d = dict(k_pages=A, v_pages=A, num_pages=8, page_size=16, num_kv_heads=2, head_dim=128, dtype=L.F16)
    return L.PagedKV(**{**d, **c})


def batch(**c):
    d = dict(page_table=A, q_starts=A, kv_lens=A, num_seqs=3, table_width=4, num_rows=10, max_q_len=5,
             max_kv_len=64)
    return L.PagedBatchDesc(**{**d, **c})


SHARED = [(dict(dtype=L.F32), {}, L.EUNSUPPORTED), (dict(head_dim=96), {}, L.EUNSUPPORTED),
          (dict(page_size=8), {}, L.EUNSUPPORTED), (dict(page_size=48), {}, L.EUNSUPPORTED),
          (dict(page_size=2048), {}, L.EUNSUPPORTED), (dict(num_pages=0), {}, L.EINVAL),
          (dict(num_kv_heads=0), {}, L.EINVAL), (dict(k_pages=None), {}, L.EINVAL),
          (dict(v_pages=A + 8), {}, L.EINVAL), ({}, dict(num_seqs=0), L.EINVAL),
          ({}, dict(num_seqs=65536), L.EINVAL), ({}, dict(table_width=0), L.EINVAL),
          ({}, dict(num_rows=0), L.EINVAL), ({}, dict(num_rows=(1 << 24) + 1), L.EINVAL),
          ({}, dict(max_q_len=0), L.EINVAL), ({}, dict(max_q_len=11), L.EINVAL),
          ({}, dict(max_kv_len=0), L.EINVAL), ({}, dict(max_kv_len=65), L.EINVAL),
          ({}, dict(page_table=None), L.EINVAL), ({}, dict(kv_lens=A + 2), L.EINVAL)]


def _append(h, k={}, b={}, ptr={}, **p):
    d = dict(num_query_heads=4, q_stride=512, k_stride=256, v_stride=256, q_out_stride=512, rotary_dim=128,
             rope_theta=1e4, eps=1e-6)
    at = {**dict(q=A, k=A, v=A, q_out=2 * A), **ptr}
    what = C.c_char_p()
    return h.h_append(C.byref(kv(**k)), C.byref(batch(**b)), *(C.c_void_p(at[n]) for n in ("q", "k", "v", "q_out")),
                      C.byref(L.PagedAppendParams(**{**d, **p})), C.byref(what)), what.value


def _attn(h, k={}, b={}, ptr={}, **p):
    d = dict(num_query_heads=4, q_stride=512, out_stride=512)
    at = {**dict(q=A, out=2 * A, lse=A), **ptr}
    what = C.c_char_p()
    return h.h_attn(C.byref(kv(**k)), C.byref(batch(**b)), *(C.c_void_p(at[n]) for n in ("q", "out", "lse")),
                    C.byref(L.PagedAttnParams(**{**d, **p})), C.byref(what)), what.value


@pytest.mark.parametrize("k,b,code", SHARED)
def test_cache_and_batch_are_checked(h, k, b, code):
    for call in (_append, _attn):
        rc, what = call(h, k, b)
        assert rc == code and what


def test_sound_arguments_pass(h):
    assert _append(h) == (L.OK, b"") and _attn(h) == (L.OK, b"")
    assert _append(h, ptr=dict(q_out=A))[0] == L.OK      # in place
    assert _append(h, num_query_heads=3)[0] == L.OK      # the append groups no heads
    assert _append(h, rotary_dim=0, rope_theta=0.)[0] == L.OK
    assert _append(h, inv_freq=A, rope_theta=0.)[0] == L.OK
    assert _attn(h, ptr=dict(lse=None))[0] == L.OK


@pytest.mark.parametrize("p,code", [
    (dict(num_query_heads=0), L.EINVAL), (dict(q_stride=504), L.EINVAL), (dict(q_stride=516), L.EINVAL),
    (dict(k_stride=248), L.EINVAL), (dict(v_stride=0), L.EINVAL), (dict(q_out_stride=0), L.EINVAL),
    (dict(rotary_dim=136), L.EUNSUPPORTED), (dict(rotary_dim=24), L.EUNSUPPORTED),
    (dict(rotary_dim=144), L.EUNSUPPORTED), (dict(rope_halves=2), L.EINVAL), (dict(rope_theta=0.), L.EINVAL),
    (dict(rope_theta=float("nan")), L.EINVAL), (dict(eps=-1.), L.EINVAL), (dict(eps=float("nan")), L.EINVAL),
    (dict(q_scale=A + 4), L.EINVAL), (dict(inv_freq=A + 4), L.EINVAL)])
def test_append_parameters_are_checked(h, p, code):
    assert _append(h, **p)[0] == code


@pytest.mark.parametrize("n,at", [("q", None), ("k", None), ("v", A + 2), ("q_out", A + 8)])
def test_append_buffers_are_checked(h, n, at):
    assert _append(h, ptr={n: at})[0] == L.EINVAL


def test_append_in_place_needs_one_stride(h):
    assert _append(h, ptr=dict(q_out=A), q_out_stride=1024)[0] == L.EINVAL


@pytest.mark.parametrize("p", [
    dict(num_query_heads=3), dict(num_query_heads=0), dict(num_query_heads=2048), dict(q_stride=256),
    dict(out_stride=513), dict(scale=-1.), dict(scale=float("inf")), dict(softcap=-1.),
    dict(softcap=float("nan")), dict(softcap=1e-30), dict(softcap=1e7), dict(scale=1e-38), dict(scale=2e30),
    dict(scale=float("nan")), dict(slopes=A + 1), dict(prefix_lens=A + 2)])
def test_attention_parameters_are_checked(h, p):
    assert _attn(h, **p)[0] == L.EINVAL


@pytest.mark.parametrize("at", [dict(q=None), dict(out=None), dict(out=A), dict(lse=A + 1), dict(q=A + 4)])
def test_attention_buffers_are_checked(h, at):
    assert _attn(h, ptr=at)[0] == L.EINVAL


@pytest.mark.parametrize("p,at,code", [
    ({}, {}, L.OK), (dict(rows=0), {}, L.EINVAL), (dict(vocab=0), {}, L.EINVAL), (dict(row_stride=99), {}, L.EINVAL),
    (dict(top_n=65, vocab=200, row_stride=200), {}, L.EINVAL), (dict(top_n=101), {}, L.EINVAL),
    (dict(vocab=4, top_n=5), {}, L.EINVAL), (dict(dtype=3), {}, L.EINVAL), (dict(temperature=0.), {}, L.EINVAL),
    (dict(temperature=float("nan")), {}, L.EINVAL), (dict(temperature=float("inf")), {}, L.EINVAL),
    (dict(temperature=1e-38), {}, L.EINVAL), (dict(temperature=-1.), {}, L.EINVAL), (dict(rows=1 << 24), {}, L.EINVAL),
    (dict(vocab=(1 << 28) + 1, row_stride=1 << 29), {}, L.EINVAL), ({}, dict(x=A + 2), L.EINVAL),
    (dict(dtype=L.F16), dict(x=A + 2), L.OK), ({}, dict(lp=None), L.EINVAL), ({}, dict(tokens=None), L.EINVAL),
    (dict(top_n=3), dict(ids=None, top=None), L.EINVAL), (dict(top_n=3), dict(ids=None), L.OK)])
def test_logprobs_arguments_are_checked(h, p, at, code):
    d = {**dict(row_stride=100, rows=2, vocab=100, top_n=0, dtype=L.F32, temperature=1.), **p}
    a = {**dict(x=A, tokens=A, lp=A, ids=A, top=A), **at}
    what = C.c_char_p()
    rc = h.h_logprobs(*(C.c_void_p(a[n]) for n in ("x", "tokens", "lp", "ids", "top")),
                      C.byref(L.LogprobsDims(**d)), C.byref(what))
    assert rc == code and bool(what.value) == (code != L.OK)


def test_null_context_and_workspace_size_need_no_gpu():
    lib = L.lib()
    assert lib.nnz_dispatch_paged_append(None, None, None, None, None, None, None, None) == L.EINVAL
    assert lib.nnz_dispatch_paged_attention(None, None, None, None, None, None, None, 0, None) == L.EINVAL
    assert lib.nnz_dispatch_token_logprobs(None, None, None, None, None, None, None, None, None, None, 0,
                                           None) == L.EINVAL
    assert lib.nnz_paged_attention_workspace_bytes(None, None, 4) == 0
    assert lib.nnz_paged_attention_workspace_bytes(C.byref(kv(head_dim=96)), C.byref(batch()), 4) == 0


def test_struct_layouts(h):
    """The same numbers are asserted of the C structs where paged_host.cc is compiled."""
    for t, size, field, at in ((L.PagedKV, 40, "dtype", 32), (L.PagedBatchDesc, 48, "max_kv_len", 40),
                               (L.PagedAppendParams, 64, "eps", 56), (L.PagedAttnParams, 40, "softcap", 36),
                               (L.LogprobsDims, 32, "temperature", 24)):
        assert C.sizeof(t) == size and getattr(t, field).offset == at


# ------------------------------------------------------------ index arithmetic
def _random_arrays(r, honest):
    seqs, width, shift = r.randint(1, 6), r.randint(1, 9), r.choice([4, 5, 6])
    max_kv = r.randint(1, width << shift)
    n = [r.randint(0, min(30, max_kv)) for _ in range(seqs)]
    lens = [r.randint(m, max_kv) for m in n]
    starts = [0]
    for m in n:
        starts.append(starts[-1] + m)
    rows = max(1, starts[-1] + r.randint(0, 3))
    max_q = max(1, max(n))
    if not honest:
        junk = [0, 1, 7, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1]
        starts = [r.choice(junk + [x]) for x in starts]
        lens = [r.choice(junk + [x]) for x in lens]
        max_q = r.randint(1, rows)
    return seqs, width, shift, rows, max_q, max_kv, starts, lens


def test_sequences_groups_and_rows_stay_in_bounds(h):
    """Over honest and broken arrays: every row a group names lies in the
    buffers, stands in that group at a position below the cache's end, and
    honest arrays' rows at positions >= 0 are each named exactly once."""
    r = random.Random(1)
    for case in range(3000):
        honest = case % 2 == 0
        seqs, width, shift, rows, max_q, max_kv, starts, lens = _random_arrays(r, honest)
        n = u32s(seqs, width, rows, max_q, max_kv, 5, shift)
        st, le = u32s(*starts), u32s(*lens)
        for s in range(seqs):
            out = (C.c_int64 * 4)()
            h.h_seq(st, le, n, s, out)
            row0, m, ln, first = out
            assert 0 <= row0 and row0 + m <= rows and 0 <= ln <= max_kv and first == ln - m
            if honest:
                assert (row0, m, ln) == (starts[s], starts[s + 1] - starts[s], lens[s])
            groups = h.h_groups(st, le, n, s)
            assert groups <= h.h_groups_max(max_q)
            named = []
            for g in range(groups):
                i = u32s(0, 0)
                h.h_group_rows(st, le, n, s, g, i)
                assert i[0] <= i[1] or i[1] == 0
                rows_of = range(i[0], i[1])
                assert len(rows_of) <= 8
                for x in rows_of:
                    assert x < min(m, max_q) and 0 <= first + x < max_kv
                    assert (first + x) // 8 == max(first, 0) // 8 + g
                named += rows_of
            assert named == [x for x in range(min(m, max_q)) if first + x >= 0]


def test_pages_out_of_range_are_none(h):
    table = u32s(0, 4, 5, 2 ** 32 - 1, 3, 1)
    n = u32s(2, 3, 1, 1, 48, 5, 4)
    got = [[h.h_page(table, n, s, j) for j in (0, 15, 16, 47, 48, 2 ** 32 - 1)] for s in (0, 1)]
    assert got == [[0, 0, 4, 5, 5, 5], [5, 5, 3, 1, 5, 5]]


def test_visible_span(h):
    def span(p, ln, prefix, window):
        out = u32s(0, 0)
        h.h_span(p, ln, prefix, window, out)
        return out[0], out[1]
    for p in (-3, -1, 0, 1, 9, 40, 2 ** 30 - 1):
        for ln in (0, 1, 10, 41, 2 ** 30):
            for prefix in (0, 5, 2 ** 32 - 1):
                for window in (0, 1, 8, 2 ** 32 - 1):
                    lo, hi = span(p, ln, prefix, window)
                    near = {j for j in range(0, 60) if j < ln and (j <= p or j < prefix)
                            and (window == 0 or j > p - window)}
                    assert {j for j in range(lo, min(hi, 60))} == near
                    assert hi <= ln


# ------------------------------------------------------------ Python's own checks
CPU = SimpleNamespace(torch_device=torch.device("cpu"), call=lambda *a: pytest.fail("reached the library"))


def _kv(num=4, heads=2, size=16, d=64, dt=torch.float16):
    return ops.PagedKVCache.empty(CPU, num, size, heads, d, dt)


def _batch(rows=6, seqs=2, width=3):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    return ops.PagedBatch(i(seqs, width), i(seqs + 1), i(seqs), rows, 3, 40)


def test_cache_tensors_are_checked():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    v = k.transpose(2, 3).contiguous()
    ops.PagedKVCache(CPU, k, v)
    for bad in ((k, k), (k, v.bfloat16()), (k.float(), v.float()), (k, k.transpose(2, 3)), (k[0], v[0])):
        with pytest.raises(NnzError):
            ops.PagedKVCache(CPU, *bad)
    with pytest.raises(NnzError):
        ops.PagedKVCache(SimpleNamespace(torch_device=torch.device("cuda", 0)), k, v)


def test_batch_tensors_are_checked():
    t, s, ln = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), \
        torch.zeros(2, dtype=torch.int32)
    ops.PagedBatch(t, s, ln, 6, 3, 40)
    for bad in ((t[0], s, ln), (t, s[:2], ln), (t, s, ln[:1]), (t.long(), s, ln), (t, s.float(), ln),
                (t.t().contiguous().t(), s, ln)):
        with pytest.raises(NnzError):
            ops.PagedBatch(*bad, 6, 3, 40)
    for bad in ((0, 3, 40), (6, -3, 40), (6, 3, 2**32 + 40)):
        with pytest.raises(NnzError):
            ops.PagedBatch(t, s, ln, *bad)


def test_rows_of_another_shape_or_type_are_refused():
    c, b = _kv(), _batch()
    q = torch.zeros(6, 4, 64, dtype=torch.float16)
    k = torch.zeros(6, 2, 64, dtype=torch.float16)
    for bad in (dict(q=q[:5]), dict(q=q.float()), dict(q_out=q.bfloat16()), dict(k=k[:, :1]),
                dict(v=torch.zeros(6, 2, 128, dtype=torch.float16)[..., ::2]), dict(q=q[0]),
                dict(q_scale=torch.ones(32)), dict(k_scale=torch.ones(64).double()),
                dict(inv_freq=torch.ones(32)), dict(inv_freq=torch.ones(64).double())):
        a = {**dict(q=q, k=k, v=k, q_out=q), **bad}
        with pytest.raises(NnzError):
            ops.dispatch_paged_append(CPU, c, b, **a)
    for bad in (dict(q=q[:, :, :32]), dict(out=q[:3]), dict(lse=torch.zeros(4, 6)), dict(slopes=torch.zeros(2)),
                dict(window=-1), dict(window=2**32 + 1),
                dict(prefix_lens=torch.zeros(2)), dict(prefix_lens=torch.zeros(3, dtype=torch.int32))):
        a = {**dict(q=q, out=q.clone(), workspace=None), **bad}
        with pytest.raises(NnzError):
            ops.dispatch_paged_attention(CPU, c, b, **a)


def test_logprobs_tensors_are_checked():
    x, i, f = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    for bad in (dict(logits=x[0]), dict(logits=x.t()), dict(logits=x.double()), dict(tokens=i.long()),
                dict(tokens=i[:2]), dict(logprobs=f.half()), dict(lse=f[:1]), dict(rank=f),
                dict(top_ids=torch.zeros(3, 4)), dict(top_ids=torch.zeros(2, 4, dtype=torch.int32)),
                dict(top_ids=torch.zeros(3, 4, dtype=torch.int32), top_logprobs=torch.zeros(3, 5))):
        with pytest.raises(NnzError):
            ops.dispatch_token_logprobs(CPU, **{**dict(logits=x, tokens=i, logprobs=f, workspace=None), **bad})
