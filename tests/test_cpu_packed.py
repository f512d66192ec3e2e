"""Host side of the packed-sequence operators: bucket tables, workspace sizes, refusals of the Python and C entry points, the
tile numbering and key ranges that the kernels derive from the lengths, and the wait states of their transfers."""
import ctypes
import math
import os
import random
import re
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import test_cpu_dma_wait_states as waits
from self_trainable_or_free_attn_amd import _lib, packed
from self_trainable_or_free_attn_amd import packed_attention, relative_buckets, shared_prefix_attention

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------ buckets
def _bucket(d, num_buckets, max_distance, bidirectional):
    """The definition, one distance at a time, in whole numbers."""
    n, first = (num_buckets // 2, num_buckets // 2 if d > 0 else 0) if bidirectional else (num_buckets, 0)
    a = abs(d) if bidirectional else max(-d, 0)
    exact = n // 2
    if a < exact:
        return first + a
    s, m = 0, n - exact
    while s + 1 < m and a ** m * exact ** (s + 1) >= max_distance ** (s + 1) * exact ** m:
        s += 1
    return first + exact + s


@pytest.mark.parametrize("num_buckets, max_distance, both", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 5, False),
                                                             (6, 40, True), (320, 800, False), (33, 100, False)])
def test_relative_buckets_follow_the_definition(num_buckets, max_distance, both):
    t = relative_buckets(num_buckets, max_distance, both).tolist()
    R = len(t) // 2
    assert len(t) % 2 == 1 and min(t) >= 0 and max(t) < num_buckets and R <= max_distance
    for d in range(-max_distance - 3, max_distance + 4):
        assert t[min(max(d, -R), R) + R] == _bucket(d, num_buckets, max_distance, both), d
    # no shorter table would do: the first distance of the last step is R
    assert R == 1 or t[0] != t[1]


def test_relative_buckets_stand_on_exact_borders():
    """64 distances, 32 buckets both ways: step 4 of 8 starts at 8 * 16^(4/8) = 32 exactly, step 6 at 8 * 16^(6/8) = 64."""
    t = relative_buckets(32, 128, True).tolist()
    R = len(t) // 2
    assert [t[R - d] for d in (31, 32, 63, 64)] == [11, 12, 13, 14]
    assert [t[R + d] for d in (31, 32, 63, 64)] == [27, 28, 29, 30]


@pytest.mark.parametrize("args", [(2, 128, True), (5, 128, True), (1, 128, False), (32, 8, True), (32, 16, False)])
def test_relative_buckets_refuse_what_has_no_steps(args):
    with pytest.raises(ValueError):
        relative_buckets(*args)


# ------------------------------------------------------------------ what the kernels derive from the lengths
def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def test_every_tile_has_one_number():
    """seq_of_tile and the first tile numbers floor(start * G / M) + b: each tile of each sequence, the rows behind the last
    one included, is found from exactly one number below the grid's size."""
    rng = random.Random(5)
    for _ in range(300):
        lens = [rng.choice([0, 1, rng.randint(0, 40), rng.randint(0, 900)]) for _ in range(rng.choice([1, 3, 64, 65, 130]))]
        G, M, pad = rng.choice([1, 2, 3, 5, 7, 8, 16]), rng.choice([64, 128]), rng.choice([0, 1, 700])
        B, T = len(lens), sum(lens) + pad
        start = _starts(lens) + [T]
        base = [start[b] * G // M + b for b in range(B + 1)]
        found = set()
        for w in range(T * G // M + B + 1):
            b = max(sum(x <= w for x in base) - 1, 0)
            t = w - base[b]
            rows = (start[b + 1] - start[b]) * G
            if t >= 0 and t * M < rows:
                assert (b, t) not in found
                found.add((b, t))
        assert found == {(b, t) for b in range(B + 1) for t in range(-(-(start[b + 1] - start[b]) * G // M))}


def test_tiles_in_order_of_their_work():
    """tile_of: up to 64 lists in descending order of weight, equal ones in their own order; every tile once, numbers below the
    sum of the tiles."""
    rng = random.Random(8)
    for _ in range(200):
        n = rng.choice([1, 2, 5, 64])
        tiles = [rng.choice([0, 1, rng.randint(0, 30)]) for _ in range(n)]
        weight = [rng.choice([0, 7, rng.randint(0, 1000)]) for _ in range(n)]
        base = [sum(tiles[j] for j in range(n) if weight[j] > weight[i] or (weight[j] == weight[i] and j < i))
                for i in range(n)]
        found = []
        for w in range(sum(tiles) + 3):
            hit = [i for i in range(n) if base[i] <= w < base[i] + tiles[i]]
            assert len(hit) == (w < sum(tiles))
            found += [(i, w - base[i]) for i in hit]
        assert sorted(found) == [(i, t) for i in range(n) for t in range(tiles[i])]
        heavy = [weight[i] for i, _ in found]
        assert heavy == sorted(heavy, reverse=True)


def test_range_items_fit_the_grid():
    """The items of a ranged launch (csrc/packed_fwd.hip, range_chunks and Cut, in float32 with a reciprocal that is off by up
    to 2^-23 either way) never outnumber the workgroups that the host starts, whichever chunk count is taken."""
    f = np.float32

    def parts(x, y, off):
        return np.ceil(f(x) * (f(1) / f(y) * f(1 + off)) - f(1e-5))

    rng = random.Random(6)
    for _ in range(1500):
        B, Hk, D = rng.choice([1, 2, 9, 64, 100]), rng.choice([1, 2, 3, 8, 40]), rng.choice([64, 128])
        G = rng.choice([1, 3, 8])
        lists = [(rng.choice([1, 1, rng.randint(0, 500)]), rng.choice([0, 1, rng.randint(0, 70), rng.randint(0, 90000)]))
                 for _ in range(B)]
        rows = [n * G for n, _ in lists]
        tiles, chunks = [-(-r // 128) for r in rows], [-(-m // 64) for _, m in lists]
        resident = 768 if D == 64 else 512
        inv_slots = f(Hk) / f(resident)
        total = f(sum(f(t) * f(c) for t, c in zip(tiles, chunks)))
        most = max([f(c) for t, c in zip(tiles, chunks) if t > 0], default=f(0))
        fair = max(np.ceil(total * inv_slots), f(1))
        for off in (-2.0 ** -23, 0.0, 2.0 ** -23):
            near = int(parts(most, fair, off))
            for n in range(max(near - 2, 1), near + 1):
                per = max(parts(most, n, off), fair)
                ranges = [max(parts(c, max(per, 4 if r <= 32 else 8), off), 1) for c, r in zip(chunks, rows)]
                items = int(sum(t * r for t, r in zip(tiles, ranges)))
                assert items <= sum(tiles) + resident // Hk + 1
                # every chunk lies in one of its tile's ranges [c i / r, c (i + 1) / r)
                assert all(int(r) >= 1 for r in ranges)


def test_tokens_of_a_row_tile():
    """The KV owner's token of a row within a tile (csrc/packed_bwd.hip, token_in_tile): (row + 1/2) / G in float32, rows up to
    G + 63 from the tile's first token on."""
    half, rows = np.float32(0.5), np.arange(64)
    for G in range(1, 4097):
        inv = np.float32(1) / np.float32(G)
        for first in {0, 1, G // 2, G - 1}:
            want = (first + rows) // G
            assert (((rows.astype(np.float32) + (np.float32(first) + half)) * inv).astype(np.int64) == want).all()
            assert ((((first + rows).astype(np.float32) + half) * inv).astype(np.int64) == want).all()


def test_division_by_multiplication():
    """fast_div of csrc/packed.h: mul = ceil(2^(32 + sh) / d), 2^sh < d <= 2^(sh + 1)."""
    rng = random.Random(7)
    for d in [2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17, 31, 33, 64, 100, 1000, 4095, 4096]:
        sh = 0
        while (2 << sh) < d:
            sh += 1
        mul = ((1 << (32 + sh)) + d - 1) // d
        assert mul < 1 << 32
        for x in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1] + [rng.randrange(2 ** 31) // d * d + e for _ in range(300) for e in (-1, 0)]:
            if x >= 0:
                assert (x * mul >> 32) >> sh == x // d


# ------------------------------------------------------------------ refusals
def _rows(n, H, D=64, dtype=torch.bfloat16):
    return torch.zeros(n, H, D, dtype=dtype)


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_packed_refusals():
    q, k = _rows(10, 4), _rows(10, 2)
    cu = _ints(0, 4, 10)
    with pytest.raises(ValueError, match="on the GPU"):
        packed_attention(q, k, k, cu)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        packed_attention(q.float(), k.float(), k.float(), cu)
    with pytest.raises(TypeError, match="k must be torch.bfloat16 like q"):
        packed_attention(q, k.half(), k, cu)
    with pytest.raises(ValueError, match="head dim must be 64 or 128"):
        packed_attention(_rows(10, 4, 96), _rows(10, 2, 96), _rows(10, 2, 96), cu)
    with pytest.raises(ValueError, match="q has head dim 64, k 128"):
        packed_attention(q, _rows(10, 2, 128), _rows(10, 2, 128), cu)
    with pytest.raises(ValueError, match="one shape"):
        packed_attention(q, k, k[:9], cu)
    with pytest.raises(ValueError, match="multiple"):
        packed_attention(q, _rows(10, 3), _rows(10, 3), cu)
    with pytest.raises(ValueError, match="multiple"):
        packed_attention(q, _rows(10, 0), _rows(10, 0), cu)
    with pytest.raises(ValueError, match="or all"):
        packed_attention(q, k[None], k[None], cu)
    with pytest.raises(ValueError, match="go with packed"):
        packed_attention(q[None], k[None], k[None], cu)
    with pytest.raises(ValueError, match="2 sequences, k 1"):
        packed_attention(q.view(2, 5, 4, 64), k[None], k[None])
    with pytest.raises(ValueError, match="cu_k needs cu_q"):
        packed_attention(q, k, k, cu_k=cu)
    with pytest.raises(ValueError, match="without cu_k"):
        packed_attention(q, _rows(11, 2), _rows(11, 2), cu)
    with pytest.raises(TypeError, match="cu_q must be int32"):
        packed_attention(q, k, k, cu.long())
    with pytest.raises(ValueError, match="contiguous"):
        packed_attention(q, k, k, _ints(0, 1, 4, 5, 10, 10)[::2])
    with pytest.raises(ValueError, match="at least two"):
        packed_attention(q, k, k, _ints(0))
    with pytest.raises(ValueError, match="cu_k must hold 3"):
        packed_attention(q, k, k, cu, _ints(0, 10))
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, k, k, cu, scale=scale)


def test_packed_bias_refusals():
    q, k, cu = _rows(10, 4), _rows(10, 2), _ints(0, 4, 10)
    t = relative_buckets(8, 20)
    w = torch.zeros(8, 4)
    with pytest.raises(ValueError, match="go together"):
        packed_attention(q, k, k, cu, bias=w)
    with pytest.raises(ValueError, match="go together"):
        packed_attention(q, k, k, cu, buckets=t)
    with pytest.raises(ValueError, match="num_buckets, 4"):
        packed_attention(q, k, k, cu, bias=w[:, :3], buckets=t)
    with pytest.raises(ValueError, match="floating-point"):
        packed_attention(q, k, k, cu, bias=w.int(), buckets=t)
    with pytest.raises(ValueError, match="2 R"):
        packed_attention(q, k, k, cu, bias=w, buckets=t[:-1].contiguous())
    with pytest.raises(TypeError, match="int32"):
        packed_attention(q, k, k, cu, bias=w, buckets=t.long())
    with pytest.raises(ValueError, match="at most 784"):
        packed_attention(q, k, k, cu, bias=w, buckets=torch.zeros(393, dtype=torch.int32))
    with pytest.raises(ValueError, match="on the GPU"):     # 2 heads a group, 391 distances: 782
        packed_attention(q, k, k, cu, bias=w, buckets=torch.zeros(391, dtype=torch.int32))


def test_shared_prefix_refusals():
    q, kp, k, lens = _rows(6, 4).view(3, 2, 4, 64), _rows(5, 2), _rows(21, 2).view(3, 7, 2, 64), _ints(1, 7, 0)
    with pytest.raises(ValueError, match="on the GPU"):
        shared_prefix_attention(q, kp, kp, k, k, lens)
    with pytest.raises(ValueError, match=r"q must be \[B, n, H, D\]"):
        shared_prefix_attention(q[0], kp, kp, k, k, lens)
    with pytest.raises(ValueError, match="k and v must have one shape"):
        shared_prefix_attention(q, kp, kp, k, k[:, :5], lens)
    with pytest.raises(ValueError, match="k_prefix and v_prefix"):
        shared_prefix_attention(q, kp, kp[:4], k, k, lens)
    with pytest.raises(ValueError, match="do not go together"):
        shared_prefix_attention(q[:2], kp, kp, k, k, lens)
    with pytest.raises(ValueError, match="do not go together"):
        shared_prefix_attention(q, _rows(5, 1), _rows(5, 1), k, k, lens)
    with pytest.raises(TypeError, match="lens must be int32"):
        shared_prefix_attention(q, kp, kp, k, k, lens.long())
    with pytest.raises(ValueError, match="lens must hold 3"):
        shared_prefix_attention(q, kp, kp, k, k, lens[:2])
    with pytest.raises(TypeError, match="v must be"):
        shared_prefix_attention(q, kp, kp, k, k.half(), lens)
    with pytest.raises(ValueError, match="k must be contiguous"):
        shared_prefix_attention(q, kp, kp, _rows(24, 2).view(3, 8, 2, 64)[:, :7], k, lens)
    with pytest.raises(ValueError, match="no backward"):
        shared_prefix_attention(q.clone().requires_grad_(), kp, kp, k, k, lens)


def _c(name, *args):
    """Status and message of a C entry point; pointers are placeholders that a refused call never follows."""
    so = _lib.lib()
    return getattr(so, name)(*args, ctypes.c_void_p(0)), so.es_last_error_string().decode()


def test_c_entry_points_refuse_before_any_launch():
    p, big = ctypes.c_void_p(256), 1 << 40

    def fwd(q=p, k=p, cu_q=p, cu_k=p, bias=None, buckets=None, nb=0, R=0, out=p, ws=p, wsb=big, B=1, Tq=8, Tk=2048, H=4, Hk=2,
            D=64, scale=1.0, suffix=""):
        return _c("es_packed_fwd" + suffix, q, k, k, cu_q, cu_k, bias, buckets, nb, R, out, out, ws, wsb, B, Tq, Tk, H, Hk, D,
                  0, scale)

    def bwd(dout=p, dq=p, dk=p, bias=None, dbias=None, ws=p, wsb=big, Tq=8, R=0, B=1, Hk=2):
        return _c("es_packed_bwd", p, p, p, dout, p, p, p, p, bias, bias, 4, R, dq, dk, dk, dbias, ws, wsb, B, Tq, 9, 4, Hk, 64,
                  0, 1.0)

    def shared(q=p, kp=p, k=p, lens=p, out=p, ws=p, wsb=big, B=2, n=1, P=9, S=5, H=4, Hk=2, D=128, scale=1.0):
        return _c("es_shared_prefix_fwd", q, kp, kp, k, k, lens, out, out, ws, wsb, B, n, P, S, H, Hk, D, scale)

    for call, status, text in [
            (lambda: fwd(D=96), 2, "64 or 128"), (lambda: fwd(H=5), 1, "multiple of Hk"), (lambda: fwd(q=None), 1, "null q"),
            (lambda: fwd(k=None), 1, "null q"), (lambda: fwd(out=None), 1, "null out"), (lambda: fwd(B=0), 1, "positive"),
            (lambda: fwd(Tq=-1), 1, "not negative"), (lambda: fwd(scale=0.0), 1, "scale"),
            (lambda: fwd(scale=math.nan), 1, "scale"), (lambda: fwd(scale=math.inf), 1, "scale"),
            (lambda: fwd(cu_q=None, B=3), 1, "equal sequences"), (lambda: fwd(H=8192, Hk=8192), 2, "4096 heads"),
            (lambda: fwd(Tq=1 << 29), 2, "too many rows"), (lambda: fwd(Tk=1 << 30), 2, "too many rows"),
            (lambda: fwd(wsb=100), 1, "workspace too small"), (lambda: fwd(ws=None), 1, "workspace too small"),
            (lambda: fwd(bias=p, nb=4, R=3), 1, "needs buckets"), (lambda: fwd(bias=p, buckets=p, R=3), 1, "needs buckets"),
            (lambda: fwd(bias=p, buckets=p, nb=4, R=196), 2, "at most 784"),
            (lambda: fwd(bias=p, buckets=p, nb=4, R=1 << 30), 2, "at most 784"),
            (lambda: fwd(D=96, suffix="_f16"), 2, "64 or 128"),
            (lambda: fwd(B=1 << 22, Hk=4), 2, "too many sequences"), (lambda: bwd(B=1 << 22, Hk=4), 2, "too many sequences"),
            (lambda: shared(B=1 << 22, Hk=4), 2, "too many sequences"),
            (lambda: fwd(q=ctypes.c_void_p(264)), 1, "aligned"), (lambda: fwd(ws=ctypes.c_void_p(260)), 1, "aligned"),
            (lambda: bwd(dq=ctypes.c_void_p(258)), 1, "aligned"), (lambda: shared(k=ctypes.c_void_p(8)), 1, "aligned"),
            (lambda: bwd(dout=None), 1, "null tensor"), (lambda: bwd(dq=None), 1, "null tensor"),
            (lambda: bwd(dk=None), 1, "null tensor"), (lambda: bwd(ws=None), 1, "null tensor"),
            (lambda: bwd(bias=p), 1, "dbias goes with bias"), (lambda: bwd(dbias=p), 1, "dbias goes with bias"),
            (lambda: bwd(wsb=8), 1, "workspace too small"),
            (lambda: shared(n=0), 1, "positive"), (lambda: shared(P=-1), 1, "not negative"),
            (lambda: shared(kp=None), 1, "null"), (lambda: shared(k=None), 1, "null"), (lambda: shared(lens=None), 1, "null"),
            (lambda: shared(D=32), 2, "64 or 128"), (lambda: shared(wsb=4), 1, "workspace too small"),
            (lambda: shared(B=1 << 20, n=1 << 12), 2, "too many rows"), (lambda: shared(scale=-1.0), 1, "scale")]:
        got, message = call()
        assert got == status and text in message, (got, message, status, text)


def test_empty_calls_launch_nothing():
    p = ctypes.c_void_p(256)
    assert _c("es_packed_fwd", None, p, p, p, p, None, None, 0, 0, None, None, None, 0, 1, 0, 9, 4, 2, 64, 0, 1.0)[0] == 0


# ------------------------------------------------------------------ the ABI and the sources
def test_operators_trace_with_meta_tensors():
    """Shapes and dtypes of the written operators and of their gradient, without a GPU."""
    q = torch.empty(10, 4, 64, dtype=torch.float16, device="meta", requires_grad=True)
    k = torch.empty(12, 2, 64, dtype=torch.float16, device="meta", requires_grad=True)
    cu = torch.empty(3, dtype=torch.int32, device="meta")
    out, lse = packed_attention(q, k, k, cu, cu, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (10, 4) and lse.dtype == torch.float32
    assert out.requires_grad and not lse.requires_grad
    dq, dk = torch.autograd.grad(out, [q, k], torch.empty_like(out))
    assert dq.shape == q.shape and dk.shape == k.shape
    c = torch.empty(3, 7, 2, 64, dtype=torch.float16, device="meta")
    t = torch.empty(3, 5, 4, 64, dtype=torch.float16, device="meta")
    out, lse = shared_prefix_attention(t, k.detach(), k.detach(), c, c, cu, return_lse=True)
    assert out.shape == t.shape and lse.shape == (3, 5, 4)


def test_header_and_bindings_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "packed_hip.h")).read(), flags=re.S)
    found = re.findall(r"\b(es_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)
    assert len(found) == 9
    so = _lib.lib()
    for name, args in found:
        n = len(args.split(","))
        if "hipStream_t" in args:
            assert len(_lib.SIGNATURES[name]) + 1 == n, name
        else:
            assert len(_lib.NO_STREAM[name][0]) == n, name
        assert hasattr(so, name)
    assert int(re.search(r"ES_PACKED_BIAS_ROWS (\d+)", text).group(1)) == packed.MAX_BIAS_ROWS


@pytest.mark.skipif(not os.path.exists(waits.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("extra", [[], ["-DES_ELEM_F16"], ["-mllvm", "-amdgpu-sched-strategy=max-ilp"]])
def test_transfers_keep_their_wait_states(extra):
    sources = ["packed_fwd.hip", "packed_bwd.hip"]
    with ThreadPoolExecutor(max_workers=2) as ex:
        asms = list(ex.map(lambda s: waits._compile(s, extra), sources))
    for src, asm in zip(sources, asms):
        n = sum(1 for s in waits._instructions(asm) if s.split()[0].startswith("buffer_load") and s.endswith(" lds"))
        assert n > 40 and not waits.violations(asm), src
