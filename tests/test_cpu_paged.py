"""Host side of norms with rotation and of paged caches: rotation tables, refusals of the Python and C entry points, derivatives that
do not exist, and the bindings."""
import ctypes
import math
import os
import re

import pytest
import torch

import test_cpu_dma_wait_states as waits
from self_trainable_or_free_attn_amd import (PagedCache, _lib, append_paged, norm_rotate, paged_attention, paged_cache, paged_rows,
                                            rotary_table)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, FP = torch.bfloat16, torch.float16


def _t(*shape, dtype=BF, device="meta"):
    return torch.empty(*shape, dtype=dtype, device=device)


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def _c(bits=16, num=8, heads=2, page=16, dim=64, dtype=BF):
    return paged_cache(num, heads, dim, page_size=page, bits=bits, dtype=dtype, device="meta")


# ------------------------------------------------------------------ tables
def test_rotary_table_follows_the_definition():
    t = rotary_table(50, 32, theta=500.0)
    assert t.shape == (50, 16, 2) and t.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (49, 15), (17, 3)):
        a = p * 500.0 ** (-2 * i / 32)
        assert abs(float(t[p, i, 0]) - math.cos(a)) <= 2 ** -24 and abs(float(t[p, i, 1]) - math.sin(a)) <= 2 ** -24


def test_far_positions_are_turned_by_their_own_angle():
    t = rotary_table(1_000_001, 16)
    a = 1_000_000 * 10000.0 ** (-2 / 16)
    assert abs(float(t[-1, 1, 0]) - math.cos(a)) <= 2 ** -23


def test_rotary_table_of_a_grid():
    t = rotary_table((2, 3, 4), (16, 8, 24))
    assert t.shape == (24, 24, 2)
    for f in range(2):
        for r in range(3):
            for c in range(4):
                row = t[(f * 3 + r) * 4 + c]
                parts = [rotary_table(n, d)[p] if d % 16 == 0 else None for n, d, p in ((2, 16, f), (3, 8, r), (4, 24, c))]
                assert torch.equal(row[:8], parts[0])
                for at, d, p in ((8, 8, r), (12, 24, c)):
                    a = p * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
                    assert torch.equal(row[at:at + d // 2, 0], a.cos().float()) and torch.equal(row[at:at + d // 2, 1], a.sin().float())


@pytest.mark.parametrize("sizes, dims", [(4, 8), (4, 0), (0, 16), ((2, 3), 16), ((2, 3), (16, 15)), ((), ()), ((2, 2), (32, -16))])
def test_rotary_table_refuses(sizes, dims):
    with pytest.raises(ValueError):
        rotary_table(sizes, dims)


# ------------------------------------------------------------------ refusals
def _rotate(q=None, k=None, qw=None, kw=None, table=None, positions=None, **kw_):
    q = _t(6, 4, 64) if q is None else q
    return norm_rotate(q, _t(6, 2, 64) if k is None else k, qw, kw, table, positions, **kw_)


W = _t(64)
TABLE = _t(6, 32, 2, dtype=torch.float32)


ROTATE_REFUSED = [
    (dict(), ValueError), (dict(qw=W), ValueError), (dict(kw=W), ValueError),
    (dict(q=_t(6, 4, 64, dtype=torch.float32), table=TABLE), TypeError), (dict(k=_t(6, 2, 64, dtype=FP), table=TABLE), TypeError),
    (dict(q=_t(6, 4, 96), k=_t(6, 2, 96), table=TABLE), ValueError), (dict(k=_t(5, 2, 64), table=TABLE), ValueError),
    (dict(q=_t(6, 64), table=TABLE), ValueError), (dict(k=_t(1, 6, 2, 64), table=TABLE), ValueError),
    (dict(q=_t(6, 0, 64), table=TABLE), ValueError), (dict(q=_t(6, 4097, 64), table=TABLE), ValueError),
    (dict(qw=_t(32), kw=_t(32)), ValueError), (dict(qw=_t(64, dtype=FP), kw=W), TypeError),
    (dict(qw=_t(64, dtype=torch.float32), kw=W), TypeError), (dict(qw=_t(1, 64), kw=W), ValueError),
    (dict(table=_t(6, 32, 2)), TypeError), (dict(table=_t(6, 64, dtype=torch.float32)), ValueError),
    (dict(table=_t(6, 4, 2, dtype=torch.float32)), ValueError), (dict(table=_t(6, 40, 2, dtype=torch.float32)), ValueError),
    (dict(table=_t(6, 0, 2, dtype=torch.float32)), ValueError), (dict(table=_t(0, 32, 2, dtype=torch.float32)), ValueError),
    (dict(table=_t(5, 32, 2, dtype=torch.float32)), ValueError),                         # fewer positions than rows
    (dict(table=_t(6, 2, 32, dtype=torch.float32).transpose(1, 2)), ValueError),
    (dict(table=TABLE, positions=_t(6, dtype=torch.int64)), TypeError), (dict(table=TABLE, positions=_i(5)), ValueError),
    (dict(qw=W, kw=W, positions=_i(6)), ValueError),
    (dict(qw=W, kw=W, eps=-1e-6), ValueError), (dict(qw=W, kw=W, eps=math.nan), ValueError), (dict(qw=W, kw=W, eps=math.inf), ValueError),
]


@pytest.mark.parametrize("kw, error", ROTATE_REFUSED)
def test_norm_rotate_refuses(kw, error):
    with pytest.raises(error):
        _rotate(**kw)


def test_norm_rotate_shapes():
    q, k = _rotate(qw=W, kw=W, table=TABLE, positions=_i(6))
    assert q.shape == (6, 4, 64) and k.shape == (6, 2, 64)
    q, k = norm_rotate(_t(3, 2, 4, 64), _t(3, 2, 2, 64), table=TABLE, positions=_i(3, 2))
    assert q.shape == (3, 2, 4, 64) and k.shape == (3, 2, 2, 64)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="GPU"):
        norm_rotate(x, x, table=rotary_table(2, 64))
    cache = paged_cache(2, 2, 64, page_size=16, device="cpu")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        append_paged(cache, x, x, ints(0)[None], ints(2))
    with pytest.raises(ValueError, match="GPU"):
        paged_rows(cache, ints(0)[None], ints(2), rows=2)


@pytest.mark.parametrize("kw", [dict(dim=96), dict(page=24), dict(page=8), dict(page=8192), dict(bits=8), dict(heads=0), dict(num=-1)])
def test_paged_cache_refuses(kw):
    with pytest.raises(ValueError):
        _c(**kw)
    with pytest.raises(TypeError):
        _c(dtype=torch.float32)


def _append(cache=None, k=None, v=None, pages=None, lens=None, cu=None, **kw):
    k = _t(6, 2, 64) if k is None else k
    v = torch.empty_like(k) if v is None else v
    return append_paged(_c() if cache is None else cache, k, v, _i(3, 4) if pages is None else pages, _i(3) if lens is None else lens,
                        cu, **kw)


APPEND_REFUSED = [
    (dict(k=_t(6, 64)), ValueError), (dict(v=_t(6, 1, 64)), ValueError), (dict(v=_t(6, 2, 64, dtype=FP)), TypeError),
    (dict(k=_t(6, 4, 64)), ValueError), (dict(k=_t(6, 2, 128)), ValueError), (dict(k=_t(7, 2, 64)), ValueError),
    (dict(k=_t(6, 2, 64, dtype=FP)), TypeError),                                       # the cache is bf16
    (dict(pages=_t(3, 4, dtype=torch.int64)), TypeError), (dict(pages=_i(3)), ValueError), (dict(pages=_i(0, 4)), ValueError),
    (dict(pages=_i(4, 3).t()), ValueError), (dict(pages=_i(3, 1 << 26)), ValueError),
    (dict(lens=_i(2)), ValueError), (dict(lens=_t(3, dtype=torch.int64)), TypeError), (dict(lens=_i(6)[::2]), ValueError),
    (dict(cu=_i(3)), ValueError), (dict(cu=_t(4, dtype=torch.int64)), TypeError),
    (dict(k=_t(3, 2, 2, 64), cu=_i(4)), ValueError), (dict(k=_t(2, 3, 2, 64)), ValueError),
    (dict(q=_t(5, 4, 64)), ValueError), (dict(q=_t(6, 4, 128)), ValueError), (dict(q=_t(6, 4, 64, dtype=FP)), TypeError),
    (dict(q=_t(6, 4, 64), k_weight=W), ValueError), (dict(q=_t(6, 4, 64), q_weight=W), ValueError), (dict(q_weight=W), ValueError),
    (dict(q_weight=W, k_weight=W), ValueError), (dict(k_weight=_t(64, dtype=FP)), TypeError), (dict(k_weight=_t(32)), ValueError),
    (dict(table=_t(6, 4, 2, dtype=torch.float32)), ValueError), (dict(eps=-1.0), ValueError),
    (dict(cache=PagedCache(_t(8, 2, 16, 64), _t(8, 2, 32, 64))), ValueError),
    (dict(cache=PagedCache(_t(8, 2, 16, 64), _t(8, 2, 16, 64).transpose(1, 2).contiguous().transpose(1, 2))), ValueError),
    (dict(cache=PagedCache(_t(8, 2, 16, 64, dtype=torch.uint8), _t(8, 2, 16, 64, dtype=torch.uint8))), TypeError),
    (dict(cache=PagedCache(_t(8, 2, 24, 64), _t(8, 2, 24, 64))), ValueError),
    (dict(cache=PagedCache(_t(8, 2, 16, 68)[..., :64], _t(8, 2, 16, 68)[..., :64])), ValueError),
    (dict(cache=PagedCache(_t(1, 2, 16, 64).expand(8, 2, 16, 64), _t(1, 2, 16, 64).expand(8, 2, 16, 64))), ValueError),
    (dict(cache=_c(4)._replace(k_scales=None)), ValueError), (dict(cache=_c(4)._replace(k_scales=_t(8, 2, 16, 4, dtype=torch.uint8))), ValueError),
    (dict(cache=_c(4)._replace(v=_t(8, 2, 16, 32, dtype=torch.int8))), TypeError),
    (dict(cache=_c(4)._replace(v=_t(8, 16, 2, 32, dtype=torch.uint8).transpose(1, 2))), ValueError),
]


@pytest.mark.parametrize("kw, error", APPEND_REFUSED)
def test_append_paged_refuses(kw, error):
    with pytest.raises(error):
        _append(**kw)


def test_append_and_rows_shapes():
    assert _append() is None
    assert _append(q=_t(6, 4, 64), q_weight=W, k_weight=W, cu=_i(4)).shape == (6, 4, 64)
    assert _append(cache=_c(4), k=_t(3, 2, 2, 64), q=_t(3, 2, 6, 64)).shape == (3, 2, 6, 64)
    for cache, dtype in ((_c(), BF), (_c(4), BF), (_c(dtype=FP), FP)):
        k, v = paged_rows(cache, _i(3, 4), _i(3), _i(4), rows=7)
        assert k.shape == v.shape == (7, 2, 64) and k.dtype == v.dtype == dtype
    assert paged_rows(_c(4), _i(3, 4), _i(3), rows=6, dtype=FP)[0].dtype == FP


@pytest.mark.parametrize("kw, error", [(dict(rows=-1), ValueError), (dict(rows=7), ValueError), (dict(rows=6, dtype=torch.float32), TypeError),
                                       (dict(rows=6, dtype=FP), TypeError), (dict(rows=1 << 30), ValueError)])
def test_paged_rows_refuses(kw, error):
    with pytest.raises(error):
        paged_rows(_c(), _i(3, 4), _i(3), **kw)


def _attend(q=None, cache=None, pages=None, lens=None, cu=None, **kw):
    return paged_attention(_t(6, 4, 64) if q is None else q, _c() if cache is None else cache, _i(3, 4) if pages is None else pages,
                           _i(3) if lens is None else lens, cu, **kw)


ATTEND_REFUSED = [
    (dict(q=_t(6, 64)), ValueError), (dict(q=_t(6, 3, 64)), ValueError), (dict(q=_t(6, 0, 64)), ValueError),
    (dict(q=_t(6, 8192, 64)), ValueError), (dict(q=_t(6, 4, 128)), ValueError), (dict(q=_t(7, 4, 64)), ValueError),
    (dict(q=_t(6, 4, 64, dtype=FP)), TypeError), (dict(q=_t(6, 4, 64, dtype=torch.float32)), TypeError),
    (dict(q=_t(2, 3, 4, 64)), ValueError), (dict(q=_t(3, 2, 4, 64), cu=_i(4)), ValueError),
    (dict(pages=_t(3, 4, dtype=torch.int64)), TypeError), (dict(pages=_i(0, 4)), ValueError), (dict(lens=_i(4)), ValueError),
    (dict(cu=_i(5)), ValueError), (dict(scale=0.0), ValueError), (dict(scale=math.inf), ValueError), (dict(scale=math.nan), ValueError),
    (dict(cache=_c(4)._replace(v_scales=None)), ValueError), (dict(cache=_c(dim=128)), ValueError),
    (dict(cache=PagedCache(_t(8, 2, 16, 64), _t(8, 2, 16, 64, dtype=FP))), TypeError),
]


@pytest.mark.parametrize("kw, error", ATTEND_REFUSED)
def test_paged_attention_refuses(kw, error):
    with pytest.raises(error):
        _attend(**kw)


def test_paged_attention_shapes():
    for cache, dtype in ((_c(), BF), (_c(4), BF), (_c(4), FP)):
        out, lse = _attend(q=_t(6, 4, 64, dtype=dtype), cache=cache, cu=_i(4), return_lse=True)
        assert out.shape == (6, 4, 64) and lse.shape == (6, 4) and out.dtype == dtype and lse.dtype == torch.float32
        out, lse = _attend(q=_t(3, 2, 6, 64, dtype=dtype), cache=cache, return_lse=True, causal=False)
        assert out.shape == (3, 2, 6, 64) and lse.shape == (3, 2, 6)


# ------------------------------------------------------------------ derivatives
def test_derivatives_that_do_not_exist_are_refused():
    k = _t(6, 2, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        _append(k=k)
    with torch.no_grad():
        _append(k=k)
    with pytest.raises(RuntimeError, match="no backward"):
        _append(k_weight=_t(64).requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        paged_rows(PagedCache(_t(8, 2, 16, 64).requires_grad_(), _t(8, 2, 16, 64)), _i(3, 4), _i(3), rows=6)
    with pytest.raises(RuntimeError, match="no backward"):
        _attend(q=_t(6, 4, 64).requires_grad_())
    with pytest.raises(RuntimeError, match="table"):
        _rotate(table=_t(6, 32, 2, dtype=torch.float32).requires_grad_())
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            _append(k=fw.make_dual(_t(6, 2, 64), _t(6, 2, 64)))


def test_the_backward_of_norm_rotate_is_not_differentiable():
    q = _t(6, 4, 64).requires_grad_()
    out, _ = _rotate(q=q, qw=W, kw=W)
    g, = torch.autograd.grad(out, q, torch.empty_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(g, q, torch.empty_like(g))


# ------------------------------------------------------------------ C ABI
def test_bindings_follow_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "paged_hip.h")).read(), flags=re.S)
    found = re.findall(r"\b(int|size_t)\s+(es_\w+)\s*\(([^)]*)\)\s*;", text)
    assert len(found) >= 13
    for kind, name, args in found:
        types = [a.rsplit(None, 1)[0].replace("*", "* ").strip() if "*" not in a else "*" for a in args.split(",")]
        want = {"*": _lib.P, "int": _lib.I, "float": _lib.F, "double": _lib.DB, "long long": _lib.LL, "size_t": _lib.Z}
        if kind == "int":
            assert types[-1] == "hipStream_t"
            assert _lib.SIGNATURES[name] == [want[t] for t in types[:-1]], name
        else:
            assert _lib.NO_STREAM[name] == ([want[t] for t in types], _lib.Z), name


P16 = ctypes.c_void_p(1 << 20)      # an aligned address that no refused call reads


def _call(name, change, base):
    args = dict(base, **change)
    return getattr(_lib.lib(), name)(*args.values(), None)


ROTATE = dict(q=P16, k=P16, qw=P16, kw=P16, table=P16, positions=None, qo=P16, ko=P16, T=4, L=4, H=4, Hk=2, D=64, R=64, P=4,
              halves=0, f32=0, eps=1e-6, qs=256, ks=128)


@pytest.mark.parametrize("change", [dict(D=96), dict(D=0), dict(T=-1), dict(H=-1), dict(H=4097), dict(q=None), dict(k=None),
                                    dict(kw=None), dict(qw=None), dict(R=8), dict(R=80), dict(R=-16), dict(R=0), dict(table=None),
                                    dict(P=0), dict(eps=-1.0), dict(eps=math.nan), dict(L=0), dict(qs=248), dict(ks=100), dict(ks=132),
                                    dict(qo=None), dict(ko=None), dict(q=ctypes.c_void_p((1 << 20) + 8)), dict(H=0),
                                    dict(T=1 << 30), dict(qo=ctypes.c_void_p((1 << 20) + 2))])
def test_c_norm_rotate_refuses_before_any_launch(change):
    for suffix in ("", "_f16"):
        assert _call("es_norm_rotate" + suffix, change, ROTATE) in (1, 2), change
        assert _lib.lib().es_last_error_string()


def test_c_norm_rotate_backward_refuses():
    base = dict(q=P16, k=P16, dqo=P16, dko=P16, qw=P16, kw=P16, table=P16, positions=None, dq=P16, dk=P16, dqw=P16, dkw=P16, ws=P16,
                bytes=1 << 20, T=4, L=4, H=4, Hk=2, D=64, R=64, P=4, halves=0, f32=0, eps=1e-6, qs=256, ks=128)
    for change in (dict(D=32), dict(dqw=None), dict(dkw=None), dict(dq=None), dict(dko=None), dict(bytes=0), dict(ws=None), dict(L=0),
                   dict(ks=8)):
        for suffix in ("", "_f16"):
            assert _call("es_norm_rotate_bwd" + suffix, change, base) in (1, 2), change


CACHE = dict(B=2, T=4, max_pages=3, num=8, page=16)


def test_c_cache_calls_refuse():
    odd = ctypes.c_void_p((1 << 20) + 4)
    rows = dict(kp=P16, vp=P16, pages=P16, lens=P16, cu=None, k=P16, v=P16, **CACHE, Hk=2, D=64, ps=2048, hs=1024, rs=64)
    rows4 = dict(kc=P16, ks=P16, vc=P16, vs=P16, pages=P16, lens=P16, cu=None, k=P16, v=P16, **CACHE, Hk=2, D=64)
    append = dict(q=P16, k=P16, v=P16, qw=P16, kw=P16, table=P16, pages=P16, lens=P16, cu=None, qo=P16, kp=P16, vp=P16, **CACHE, H=4,
                  Hk=2, D=64, R=64, P=4, halves=0, f32=0, eps=1e-6, qs=256, kst=128, vst=128, ps=2048, hs=1024, rs=64)
    append4 = {n: x for n, x in append.items() if n not in ("ps", "hs", "rs", "kp", "vp")}
    at = list(append4).index("B")
    items = list(append4.items())
    append4 = dict(items[:at] + [("kc", P16), ("ks", P16), ("vc", P16), ("vs", P16)] + items[at:])
    common = [dict(B=0), dict(T=5), dict(T=-1), dict(page=24), dict(page=8), dict(page=8192), dict(max_pages=1 << 26), dict(lens=None),
              dict(pages=None), dict(D=96), dict(Hk=0), dict(num=-1), dict(max_pages=-1), dict(B=1 << 24, T=1 << 24)]
    fwd = dict(q=P16, kp=P16, vp=P16, pages=P16, lens=P16, cu=None, out=P16, lse=P16, ws=P16, bytes=1 << 30, **CACHE, H=4, Hk=2, D=64,
               causal=1, scale=0.1, ps=2048, hs=1024, rs=64)
    fwd4 = dict(q=P16, kc=P16, ks=P16, vc=P16, vs=P16, pages=P16, lens=P16, cu=None, out=P16, lse=P16, ws=P16, bytes=1 << 30, **CACHE,
                H=4, Hk=2, D=64, causal=1, scale=0.1)
    attend = [dict(H=5), dict(H=0), dict(H=8194), dict(q=None), dict(out=None), dict(lse=None), dict(out=odd), dict(q=odd), dict(scale=0.0),
              dict(scale=math.nan), dict(max_pages=4096, ws=None), dict(max_pages=4096, bytes=64)]
    for name, base, more in (
            ("es_paged_fwd", fwd, attend + [dict(kp=None), dict(vp=odd), dict(rs=32)]),
            ("es_paged4_fwd", fwd4, attend + [dict(kc=None), dict(vs=None), dict(ks=odd)]),
            ("es_paged_rows", rows, [dict(kp=None), dict(vp=odd), dict(rs=60), dict(rs=32), dict(hs=-8), dict(ps=4), dict(k=None),
                                     dict(v=odd), dict(rs=1 << 30)]),
            ("es_paged_rows4", rows4, [dict(kc=None), dict(vs=None), dict(ks=odd), dict(k=None)]),
            ("es_append_paged", append, [dict(kp=None), dict(rs=60), dict(qo=None), dict(v=None), dict(qs=8), dict(vst=130), dict(R=8),
                                         dict(kw=None), dict(H=-1)]),
            ("es_append_paged4", append4, [dict(kc=None), dict(vs=odd), dict(qo=None), dict(v=odd), dict(kst=64), dict(P=0)])):
        assert len(base) == len(_lib.SIGNATURES[name]), name
        for change in common + more:
            for suffix in ("", "_f16"):
                assert _call(name + suffix, change, base) in (1, 2), (name, change)
    # nothing to do: no launch, no error
    for name, base in (("es_paged_fwd", fwd), ("es_paged4_fwd", fwd4), ("es_paged_rows", rows), ("es_paged_rows4", rows4), ("es_append_paged", append), ("es_append_paged4", append4)):
        assert _call(name, dict(T=0), base) == 0


def test_direct_operator_calls_check_their_tensors():
    ops = _lib.ops()
    x = torch.zeros(2, 2, 64, dtype=BF)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.norm_rotate(x, x, None, None, rotary_table(2, 64), None, 2, False, 1e-6)


# ------------------------------------------------------------------ transfers into LDS
@pytest.mark.skipif(not os.path.exists(waits.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("extra", [[], ["-DES_ELEM_F16"], ["-mllvm", "-amdgpu-sched-strategy=max-ilp"]])
def test_transfers_keep_their_wait_states(extra):
    asm = waits._compile("paged_fwd.hip", extra)
    n = sum(1 for s in waits._instructions(asm) if s.split()[0].startswith("buffer_load") and s.endswith(" lds"))
    assert n > 40 and not waits.violations(asm)
