"""The bounded KV cache on the GPU against its formulas in 64 bits (on the CPU): the normalised and rotated store, the attention with the
weight every slot draws, the eviction, and the three run one after the other as a decode loop does."""
import math

import numpy as np
import pytest
import torch

import llm_amd.blocks as B
import llm_amd.kernels as K
import llm_amd.ops as ops

pytestmark = pytest.mark.gpu

U32, U16, UBF = 2.0 ** -24, 2.0 ** -11, 2.0 ** -8          # half a step relative to the value: f32, f16, bf16
DTYPE = {B.F32: torch.float32, B.F16: torch.float16, B.BF16: torch.bfloat16}


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def values(rows, t):
    """f64 values of cache rows (CPU tensor)"""
    if t in DTYPE:
        return rows.double()
    b = rows.reshape(*rows.shape[:-1], -1, B.TYPE_SIZE[t])
    d = b[..., :2].contiguous().view(torch.float16).double()
    q = b[..., 2:].contiguous()
    q = q.view(torch.int8).double() if t == B.Q8_0 else torch.cat([q & 15, q >> 4], -1).double() - 8
    return (d * q).reshape(*rows.shape[:-1], -1)


def cache(shape, t, g, scale=1.0):
    """random cache rows of type t (CPU)"""
    if t in DTYPE:
        return (torch.randn(shape, generator=g) * scale).to(DTYPE[t])
    n = math.prod(shape[:-1])
    return torch.from_numpy(B.random_blocks(t, n, shape[-1], seed=int(torch.randint(0, 1 << 30, (1,), generator=g)),
                                            scale=scale * (0.02 if t == B.Q8_0 else 0.3))).reshape(*shape[:-1], -1)


# ---- qk_norm_rope --------------------------------------------------------------------------------------------------------------------

def store_oracle(x, w, eps, pos, n_dims, mode, base=10000.0, ff=None, freq_scale=1.0, ext=0.0, attn=1.0, n_ctx=8192, fast=32.0, slow=1.0):
    """-> (values, per value a bound of its f32 error) of rope(rms_norm(x) * w), x [S, n, H, d] -> [S, H, n, d]"""
    x = x.double()
    d = x.shape[-1]
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() if w is not None else 1.0)
    # the sum of squares: at most d / 64 + 8 additions deep in any of the kernels' trees (16 lanes x 8 values); root, quotient, two products
    err = y.abs() * (24 * U32)
    if n_dims:
        i = torch.arange(n_dims // 2, dtype=torch.float64)
        f = base ** (-2.0 * i / n_dims) / (ff.double() if ff is not None else 1.0)
        if ext != 0.0:
            dim = lambda rot: n_dims * math.log(n_ctx / (rot * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(0, math.floor(dim(fast))), min(n_dims - 1, math.ceil(dim(slow)))
            mix = (1 - torch.clamp((i - lo) / max(0.001, hi - lo), 0, 1)) * ext
            f = f * (freq_scale * (1 - mix) + mix)
            attn *= 1 + 0.1 * math.log(1 / freq_scale)
        else:
            f = f * freq_scale
        t = pos.double()[:, :, None, None] * f
        r, keep = y[..., :n_dims], y[..., n_dims:]
        a, b = (r[..., 0::2], r[..., 1::2]) if mode == 0 else (r[..., : n_dims // 2], r[..., n_dims // 2:])
        c, s = torch.cos(t) * attn, torch.sin(t) * attn
        u, v = a * c - b * s, a * s + b * c
        # the norm's 24, the angle rounded to f32 revolutions (2 pi 2^-26 of a turn), sincos (4 steps of 2^-24), products and sum (3)
        e = torch.hypot(a, b) * (36 * U32 * max(1.0, abs(attn)))
        # f32 parameters of YaRN (the ramp's ends, freq_scale): relative 2^-23 of the angle
        if ext != 0.0 or freq_scale != 1.0:
            e = e + torch.hypot(a, b) * (t.abs() * 2.0 ** -22 + 2.0 ** -22)
        if mode == 0:
            y, err = torch.cat([torch.stack([u, v], -1).flatten(-2), keep], -1), torch.cat([torch.stack([e, e], -1).flatten(-2), err[..., n_dims:]], -1)
        else:
            y, err = torch.cat([u, v, keep], -1), torch.cat([e, e, err[..., n_dims:]], -1)
    return y.transpose(1, 2), err.transpose(1, 2)


def store_case(S, n, H, HK, d, dv, slots, t, seed, layout="dense"):
    g = gen(seed)
    mk = lambda h, m: torch.randn((S, n, h, m), generator=g) * 3  # noqa: E731
    q, k, v = mk(H, d), mk(HK, d), mk(HK, dv)
    dev = dict(q=q.cuda(), k=k.cuda(), v=v.cuda())
    if layout == "packed":                       # one row of q, k and v heads per token, as a fused projection leaves it
        both = torch.cat([x.reshape(S, n, -1) for x in (q, k, v)], -1).cuda()
        off = 0
        for name, h, m in (("q", H, d), ("k", HK, d), ("v", HK, dv)):
            dev[name] = both[..., off:off + h * m].unflatten(-1, (h, m))
            off += h * m
    qw, kw = 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
    rows = torch.stack([torch.randperm(slots, generator=g)[:n] for _ in range(S * HK)]).reshape(S, HK, n).to(torch.int32)
    kc, vc = cache((S, HK, slots, d), t, g), cache((S, HK, slots, dv), t, g)
    pos = torch.randint(0, 200000, (S, n), generator=g).to(torch.int32)
    return q, k, v, dev, qw, kw, rows, kc, vc, pos


def check_rows(got, before, rows, want, err, t):
    """stored rows hold the values (rounded once), every other row its bytes of before"""
    S, HK, slots = before.shape[:3]
    at = (torch.arange(S)[:, None, None], torch.arange(HK)[None, :, None], rows.long())
    touched = torch.zeros((S, HK, slots), dtype=torch.bool)
    touched[at] = True
    assert torch.equal(got[~touched].view(torch.uint8) if got.dtype != torch.uint8 else got[~touched],
                       before[~touched].view(torch.uint8) if before.dtype != torch.uint8 else before[~touched])
    u = {B.F32: 0.0, B.F16: U16, B.BF16: UBF}[t]
    x = got[at].double()
    # once rounded; below the normal range of f16 half a step is 2^-25
    assert ((x - want).abs() <= err + u * (want.abs() + err) + (2.0 ** -25 if t == B.F16 else 0.0)).all()


STORE = [
    # S, n, H, HK, d, dv, slots, type, n_dims, mode, layout
    (1, 1, 32, 8, 128, 128, 64, B.F16, 128, 2, "dense"),
    (1, 1, 32, 8, 128, 128, 64, B.F16, 128, 0, "packed"),
    (3, 1, 64, 8, 128, 128, 9, B.BF16, 128, 2, "dense"),
    (1, 37, 8, 2, 64, 64, 50, B.F32, 64, 2, "packed"),
    (2, 5, 5, 5, 80, 80, 7, B.F16, 40, 2, "dense"),
    (1, 130, 4, 1, 96, 64, 131, B.BF16, 48, 0, "dense"),
    (1, 7, 3, 1, 256, 256, 7, B.F16, 256, 2, "packed"),
    (2, 3, 2, 1, 256, 128, 4, B.F32, 64, 0, "dense"),
    (1, 2, 1, 1, 8, 8, 3, B.F16, 8, 2, "dense"),
    (1, 9, 6, 3, 72, 40, 11, B.F16, 72, 0, "dense"),
    (1, 4, 4, 2, 128, 128, 5, B.F16, 0, 2, "dense"),
    (1, 600, 16, 2, 128, 128, 600, B.F16, 128, 2, "dense"),
]


@pytest.mark.parametrize("S,n,H,HK,d,dv,slots,t,n_dims,mode,layout", STORE)
def test_store_against_the_formula(S, n, H, HK, d, dv, slots, t, n_dims, mode, layout):
    q, k, v, dev, qw, kw, rows, kc, vc, pos = store_case(S, n, H, HK, d, dv, slots, t, 17 + n + d, layout)
    kg, vg = kc.cuda(), vc.cuda()
    sp, sm = torch.full((S, HK, slots), 7, dtype=torch.int32, device="cuda"), torch.full((S, HK, slots), 3.0, device="cuda")
    qo = ops.qk_norm_rope(dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kg, vg, t, rows=rows.cuda(), slot_pos=sp, slot_mass=sm,
                          n_dims=n_dims, mode=mode, freq_base=500000.0)
    want, err = store_oracle(q, qw, 1e-6, pos, n_dims, mode, base=500000.0)
    assert ((qo.cpu().double() - want).abs() <= err).all()
    check_rows(kg.cpu(), kc, rows, *store_oracle(k, kw, 1e-6, pos, n_dims, mode, base=500000.0), t)
    check_rows(vg.cpu(), vc, rows, v.double().transpose(1, 2), torch.zeros(()), t)
    at = (torch.arange(S)[:, None, None], torch.arange(HK)[None, :, None], rows.long())
    wp, wm = torch.full((S, HK, slots), 7, dtype=torch.int32), torch.full((S, HK, slots), 3.0)
    wp[at], wm[at] = pos[:, None, :].expand(S, HK, n), 0.0
    assert torch.equal(sp.cpu(), wp) and torch.equal(sm.cpu(), wm)


@pytest.mark.parametrize("t", [B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("d,dv,n_dims,mode", [(128, 128, 128, 2), (64, 96, 64, 0), (96, 32, 40, 2), (256, 256, 64, 2), (32, 32, 8, 0)])
def test_store_into_blocks_quantizes_the_rotated_rows(t, d, dv, n_dims, mode):
    """the f32 rows of the same call, quantized by SET_ROWS: the same bytes"""
    S, n, H, HK, slots = 2, 11, 4, 2, 12
    q, k, v, dev, qw, kw, rows, kc, vc, pos = store_case(S, n, H, HK, d, dv, slots, t, d + n_dims)
    v[0, 0, 0, :32] = 0.0
    dev["v"] = v.cuda()
    kg, vg = kc.cuda(), vc.cuda()
    args = (dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda())
    qo = ops.qk_norm_rope(*args, kg, vg, t, rows=rows.cuda(), n_dims=n_dims, mode=mode)
    kf, vf = torch.zeros((S, HK, slots, d), device="cuda"), torch.zeros((S, HK, slots, dv), device="cuda")
    qf = ops.qk_norm_rope(*args, kf, vf, B.F32, rows=rows.cuda(), n_dims=n_dims, mode=mode)
    assert torch.equal(qo, qf)
    for got, src, before in ((kg, kf, kc), (vg, vf, vc)):
        all_rows = torch.arange(slots, dtype=torch.int64, device="cuda")
        blocks = torch.zeros_like(got)
        for s in range(S):
            for h in range(HK):
                ops.set_rows(src[s, h].contiguous(), all_rows, blocks[s, h], t)
        at = (torch.arange(S)[:, None, None], torch.arange(HK)[None, :, None], rows.long())
        want = before.clone()
        want[at] = blocks.cpu()[at]
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("mode", [0, 2])
def test_store_with_yarn_and_frequency_factors(mode):
    q, k, v, dev, qw, kw, rows, kc, vc, pos = store_case(1, 6, 4, 2, 128, 128, 8, B.F32, 5)
    pos = torch.tensor([[0, 1, 77, 4096, 30000, 131071]], dtype=torch.int32)
    ff = 1 + torch.rand(64, generator=gen(3)) * 7
    kw_ = dict(n_dims=128, mode=mode, freq_base=1e6, freq_scale=0.25, ext_factor=1.0, attn_factor=0.9, n_ctx_orig=32768)
    kg, vg = kc.cuda(), vc.cuda()
    qo = ops.qk_norm_rope(dev["q"], dev["k"], dev["v"], qw.cuda(), None, 1e-5, pos.cuda(), kg, vg, B.F32, rows=rows.cuda(), freq_factors=ff.cuda(), **kw_)
    o = dict(base=1e6, ff=ff, freq_scale=0.25, ext=1.0, attn=0.9, n_ctx=32768)
    want, err = store_oracle(q, qw, 1e-5, pos, 128, mode, **o)
    assert ((qo.cpu().double() - want).abs() <= err).all()
    check_rows(kg.cpu(), kc, rows, *store_oracle(k, None, 1e-5, pos, 128, mode, **o), B.F32)


def test_store_skips_rows_outside_the_cache_and_q_may_stay_in_place():
    S, n, H, HK, d, slots = 1, 5, 4, 2, 128, 6
    q, k, v, dev, qw, kw, _, kc, vc, pos = store_case(S, n, H, HK, d, d, slots, B.F16, 11)
    rows = torch.tensor([[[-1, 0, 6, 5, 2 ** 31 - 1], [3, -2 ** 31, 1, 100, 2]]], dtype=torch.int32)
    sp, sm = torch.full((S, HK, slots), 7, dtype=torch.int32, device="cuda"), torch.full((S, HK, slots), 3.0, device="cuda")
    kg, vg = kc.cuda(), vc.cuda()
    want, err = store_oracle(q, qw, 1e-6, pos, d, 2)
    qo = ops.qk_norm_rope(dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kg, vg, B.F16, rows=rows.cuda(), slot_pos=sp, slot_mass=sm,
                          q_out=dev["q"].transpose(1, 2))
    assert qo.data_ptr() == dev["q"].data_ptr() and ((qo.cpu().double() - want).abs() <= err).all()
    wk, e = store_oracle(k, kw, 1e-6, pos, d, 2)
    for h in range(HK):
        for i in range(n):
            r = int(rows[0, h, i])
            if 0 <= r < slots:
                assert ((kg[0, h, r].cpu().double() - wk[0, h, i]).abs() <= e[0, h, i] + U16 * (wk[0, h, i].abs() + e[0, h, i]) + 2.0 ** -25).all()
                assert torch.equal(vg[0, h, r].cpu(), v[0, i, h].half()) and int(sp[0, h, r]) == int(pos[0, i]) and float(sm[0, h, r]) == 0.0
        for r in set(range(slots)) - set(rows[0, h].tolist()):
            assert torch.equal(kg[0, h, r].cpu(), kc[0, h, r]) and torch.equal(vg[0, h, r].cpu(), vc[0, h, r])
            assert int(sp[0, h, r]) == 7 and float(sm[0, h, r]) == 3.0


def test_store_without_v_without_rows_of_nothing_and_of_zeros():
    q, k, _, dev, qw, kw, _, kc, _, pos = store_case(1, 3, 2, 1, 64, 64, 3, B.F16, 12)
    q[0, 1] = 0.0                                 # a row of zeros normalises to zeros
    kg = kc.cuda()
    qo = ops.qk_norm_rope(q.cuda(), dev["k"], None, qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kg, None, B.F16)
    want, err = store_oracle(q, qw, 1e-6, pos, 64, 2)
    assert ((qo.cpu().double() - want).abs() <= err).all() and (qo[0, :, 1] == 0).all()
    check_rows(kg.cpu(), kc, torch.arange(3)[None, None], *store_oracle(k, kw, 1e-6, pos, 64, 2), B.F16)
    none = torch.zeros((1, 0, 2, 64), device="cuda")
    out = ops.qk_norm_rope(none, none[:, :, :1], None, None, None, 1e-6, pos.cuda()[:, :0], kg, None, B.F16)
    assert out.shape == (1, 2, 0, 64)


@pytest.mark.parametrize("t", [B.F16, B.Q4_0])
def test_store_into_a_cache_of_no_rows(t):
    """nothing to store into: q is normalised and rotated all the same"""
    q, k, v, dev, qw, kw, _, _, _, pos = store_case(2, 3, 4, 2, 64, 64, 4, B.F16, 15)
    none = torch.zeros((2, 2, 0, 64 if t in DTYPE else 2 * B.TYPE_SIZE[t]), dtype=DTYPE.get(t, torch.uint8), device="cuda")
    want, err = store_oracle(q, qw, 1e-6, pos, 64, 2)
    for vv, vc in ((dev["v"], none), (None, None)):
        qo = ops.qk_norm_rope(dev["q"], dev["k"], vv, qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), none, vc, t)
        assert ((qo.cpu().double() - want).abs() <= err).all()


def test_store_with_rows_and_tables_that_all_heads_share():
    """one slot for every head of a token: rows with a stride of 0 over the heads, slot_pos and slot_mass expanded over them"""
    S, n, H, HK, d, slots = 2, 3, 4, 2, 64, 9
    q, k, v, dev, qw, kw, _, kc, vc, pos = store_case(S, n, H, HK, d, d, slots, B.F16, 16)
    rows = torch.stack([torch.randperm(slots, generator=gen(s))[:n] for s in range(S)]).to(torch.int32)[:, None]
    kg, vg = kc.cuda(), vc.cuda()
    sp, sm = torch.full((S, 1, slots), 7, dtype=torch.int32, device="cuda"), torch.full((S, 1, slots), 3.0, device="cuda")
    ops.qk_norm_rope(dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kg, vg, B.F16, rows=rows.cuda().expand(S, HK, n),
                     slot_pos=sp.expand(S, HK, slots), slot_mass=sm.expand(S, HK, slots))
    check_rows(kg.cpu(), kc, rows.expand(S, HK, n), *store_oracle(k, kw, 1e-6, pos, d, 2), B.F16)
    want = torch.full((S, slots), 7, dtype=torch.int32).scatter(1, rows[:, 0].long(), pos)
    assert torch.equal(sp[:, 0].cpu(), want) and torch.equal(sm[:, 0].cpu(), torch.where(want == 7, 3.0, 0.0))
    with pytest.raises(K.Mi355Error):             # a cache that the heads share is another matter
        ops.qk_norm_rope(dev["q"], dev["k"], None, None, None, 1e-6, pos.cuda(), kg[:, :1].expand(S, HK, slots, d), None, B.F16)


@pytest.mark.parametrize("t", [B.F16, B.BF16])
def test_store_into_a_pool_that_sequences_share(t):
    """one cache for all sequences (a stride of 0 over them), each token in a row of its own"""
    S, n, H, HK, d, slots = 3, 4, 4, 2, 64, 20
    q, k, v, dev, qw, kw, _, _, _, pos = store_case(S, n, H, HK, d, d, slots, t, 18)
    g = gen(19)
    rows = torch.stack([torch.randperm(slots, generator=g)[: S * n] for _ in range(HK)]).reshape(HK, S, n).transpose(0, 1).contiguous().to(torch.int32)
    kc, vc = cache((1, HK, slots, d), t, g), cache((1, HK, slots, d), t, g)
    kg, vg = kc.cuda(), vc.cuda()
    ops.qk_norm_rope(dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kg.expand(S, HK, slots, d), vg.expand(S, HK, slots, d), t, rows=rows.cuda())
    flat = lambda x: x.transpose(0, 1).reshape(1, HK, S * n, *x.shape[3:])  # noqa: E731
    want, err = store_oracle(k, kw, 1e-6, pos, d, 2)
    check_rows(kg.cpu(), kc, flat(rows), flat(want), flat(err), t)
    check_rows(vg.cpu(), vc, flat(rows), flat(v.double().transpose(1, 2)), torch.zeros(()), t)


def test_store_on_another_stream_and_captured():
    """launched on the current stream whatever it is; a captured launch reads new rows and positions at every replay"""
    S, n, H, HK, d, slots = 2, 1, 8, 2, 128, 16
    q, k, v, dev, qw, kw, rows, kc, vc, pos = store_case(S, n, H, HK, d, d, slots, B.F16, 13)
    qg, kg, vg, rg, pg, qwg, kwg = dev["q"], kc.cuda(), vc.cuda(), rows.cuda(), pos.cuda(), qw.cuda(), kw.cuda()
    qo = torch.empty((S, H, n, d), device="cuda")
    run = lambda: ops.qk_norm_rope(qg, dev["k"], dev["v"], qwg, kwg, 1e-6, pg, kg, vg, B.F16, rows=rg, q_out=qo)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    g = gen(4)
    for _ in range(4):
        rows = torch.stack([torch.randperm(slots, generator=g)[:n] for _ in range(S * HK)]).reshape(S, HK, n).to(torch.int32)
        pos = torch.randint(0, 100000, (S, n), generator=g).to(torch.int32)
        before = kg.cpu()
        rg.copy_(rows); pg.copy_(pos); qo.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, err = store_oracle(q, qw, 1e-6, pos, d, 2)
        assert ((qo.cpu().double() - want).abs() <= err).all()
        check_rows(kg.cpu(), before, rows, *store_oracle(k, kw, 1e-6, pos, d, 2), B.F16)


def test_store_wrapper_refuses_what_does_not_fit():
    q, k, v, dev, qw, kw, rows, kc, vc, pos = store_case(1, 2, 4, 2, 64, 64, 4, B.F16, 14)
    a = [dev["q"], dev["k"], dev["v"], qw.cuda(), kw.cuda(), 1e-6, pos.cuda(), kc.cuda(), vc.cuda(), B.F16]
    for i, bad in ((0, dev["q"].half()), (1, dev["k"][:, :1]), (2, None), (6, pos.cuda().long()), (7, kc.cuda().bfloat16()), (7, kc.cuda()[..., :32]),
                   (8, vc.cuda()[:, :, :3]), (3, qw), (9, B.Q4_K)):
        b = list(a)
        b[i] = bad
        with pytest.raises(ValueError):
            ops.qk_norm_rope(*b)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(*a, rows=rows.cuda().long())
    with pytest.raises(K.Mi355Error):
        ops.qk_norm_rope(*a, mode=1)
    with pytest.raises(K.Mi355Error):
        ops.qk_norm_rope(dev["q"][..., 4:36], dev["k"][..., 4:36], None, None, None, 1e-6, pos.cuda(), kc.cuda()[..., 4:36], None, B.F16)   # 8-byte aligned cache


# ---- kv_evict ------------------------------------------------------------------------------------------------------------------------

def evict_oracle(mass, pos, past, used, n_keep, n_evict, sink, recent):
    """numpy: (kept, evicted) by a stable sort of the keys"""
    S, HK, n = mass.shape
    kept, evicted = np.full((S, HK, n_keep), -1, np.int32), np.full((S, HK, n_evict), -1, np.int32)
    for s in range(S):
        u = min(max(int(used[s]), 0), n)
        for h in range(HK):
            key = mass[s, h, :u].astype(np.float64)
            key = np.where(np.isnan(key), -np.inf, key)
            p = pos[s, h, :u].astype(np.int64)
            key = np.where((p < sink) | (p >= int(past[s]) - recent), np.inf, key)
            order = np.lexsort((np.arange(u), -key))
            k, e = np.sort(order[:n_keep]), np.sort(order[n_keep:])[:n_evict]
            kept[s, h, :len(k)], evicted[s, h, :len(e)] = k, e
    return kept, evicted


def evict_case(S, HK, n, seed, kind="spread"):
    r = np.random.default_rng(seed)
    mass = (r.random((S, HK, n)) ** 6 * 20).astype(np.float32)
    if kind == "ties":
        mass = r.integers(0, 3, (S, HK, n)).astype(np.float32)
        mass[r.random(mass.shape) < 0.2] = -0.0
    elif kind == "equal":
        mass[:] = 0.25
    elif kind == "odd":                  # infinities, NaNs, negative and subnormal values, neighbours in the last bit
        pool = np.array([np.inf, -np.inf, np.nan, -np.nan, 0.0, -0.0, 1e-45, -1e-45, 1.0, np.nextafter(np.float32(1), np.float32(2)), -1.0, 3e38, -3e38], np.float32)
        mass = pool[r.integers(0, len(pool), (S, HK, n))]
    elif kind == "border":               # a few hundred keys around the border, one step of the last bit apart, some of them equal
        mass = (np.float32(1.0).view(np.uint32) + r.integers(0, 100, (S, HK, n)).astype(np.uint32)).view(np.float32)
        mass[..., ::7] = 5.0
        mass[..., 3::7] = -2.0
    pos = np.stack([r.permutation(2 * n + 3)[:n] for _ in range(S * HK)]).reshape(S, HK, n).astype(np.int32)
    return mass, pos


EVICT = [
    # S, HK, n_kv, n_keep, sink, recent, used, kind
    (1, 1, 1, 1, 0, 0, None, "spread"), (1, 2, 2, 1, 0, 0, None, "spread"), (2, 3, 65, 64, 4, 16, None, "spread"), (1, 8, 2049, 2048, 4, 512, None, "spread"),
    (3, 2, 1000, 100, 4, 25, [1000, 100, 99], "ties"), (4, 1, 777, 300, 0, 0, [0, 1, 301, 5000], "equal"), (2, 2, 500, 123, 0, 0, [-7, 500], "odd"),
    (1, 2, 4097, 17, 17, 0, None, "ties"), (1, 2, 5000, 4999, 0, 4999, None, "odd"), (1, 1, 100, 200, 10, 10, None, "spread"),
    (2, 2, 3000, 1500, 0, 0, [3000, 2999], "ties"), (1, 3, 8000, 7999, 4, 100, None, "equal"), (1, 2, 16000, 1, 0, 0, None, "spread"), (3, 1, 50000, 20000, 4, 1024, [50000, 100, 40000], "odd"),
    (2, 2, 600, 300, 0, 0, None, "border"), (1, 2, 150, 60, 0, 0, None, "border"), (1, 1, 9000, 4000, 4, 10, None, "border"), (1, 2, 40000, 17000, 4, 10, None, "border"),
    (2, 4, 32768, 4096, 4, 1024, [32768, 20001], "spread"), (1, 2, 70001, 9000, 4, 100, None, "ties"), (1, 1, 140000, 100000, 4, 100, None, "odd"),
]


@pytest.mark.parametrize("S,HK,n,n_keep,sink,recent,used,kind", EVICT)
def test_evict_picks_the_heaviest(S, HK, n, n_keep, sink, recent, used, kind):
    mass, pos = evict_case(S, HK, n, n + n_keep, kind)
    past = np.full(S, 2 * n + 3, np.int32)
    u = np.array(used if used is not None else [n] * S, np.int32)
    for n_evict in {max(0, n - n_keep), min(1, n - n_keep) if n > n_keep else 0}:
        kept, evicted = ops.kv_evict(torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda(), torch.from_numpy(past).cuda(), n_keep, sink, recent,
                                     n_used=torch.from_numpy(u).cuda() if used is not None else None, n_evict=n_evict)
        wk, we = evict_oracle(mass, pos, past, u, n_keep, n_evict, sink, recent)
        assert np.array_equal(kept.cpu().numpy(), wk) and np.array_equal(evicted.cpu().numpy(), we)


@pytest.mark.parametrize("t,d,dv", [(B.F16, 128, 128), (B.Q8_0, 128, 96), (B.Q4_0, 64, 64), (B.BF16, 72, 40), (B.F32, 256, 256), (B.F16, 1, 3)])
def test_evict_gathers_rows_as_they_are(t, d, dv):
    """rows byte for byte, tables beside them; rows behind the last kept one, and memory around the views, stay as they were"""
    S, HK, n, n_keep = 2, 3, 300, 90
    mass, pos = evict_case(S, HK, n, d + dv)
    past, u = np.full(S, 2 * n + 3, np.int32), np.array([n, 60], np.int32)
    rb = lambda m: B.row_size(t, m)  # noqa: E731
    g = gen(9)
    raw = [torch.randint(0, 256, (S, n, HK, rb(m) + 32), generator=g).to(torch.uint8).cuda() for m in (d, dv)]             # slot-major storage, padded rows
    out = [torch.full((S, HK, n_keep + 2, rb(m) + 16), 77, dtype=torch.uint8, device="cuda") for m in (d, dv)]
    view = lambda x, m: x[..., 16:16 + rb(m)] if t in (B.Q8_0, B.Q4_0) else x[..., 16:16 + rb(m)].view(DTYPE[t])  # noqa: E731
    src = [view(x, m).transpose(1, 2) for x, m in zip(raw, (d, dv))]
    dst = [(x[..., :rb(m)] if t in (B.Q8_0, B.Q4_0) else x[..., :rb(m)].view(DTYPE[t]))[:, :, :n_keep] for x, m in zip(out, (d, dv))]
    kept, evicted, mo, po = ops.kv_evict(torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda(), torch.from_numpy(past).cuda(), n_keep, 4, 20,
                                         n_used=torch.from_numpy(u).cuda(), k=src[0], v=src[1], type_kv=t, k_out=dst[0], v_out=dst[1])
    wk, _ = evict_oracle(mass, pos, past, u, n_keep, 0, 4, 20)
    assert np.array_equal(kept.cpu().numpy(), wk)
    wm, wp = np.zeros((S, HK, n_keep), np.float32), np.full((S, HK, n_keep), -1, np.int32)
    want = [torch.full_like(x.cpu(), 77) for x in out]
    for s in range(S):
        for h in range(HK):
            k = wk[s, h][wk[s, h] >= 0]
            wm[s, h, :len(k)], wp[s, h, :len(k)] = mass[s, h, k], pos[s, h, k]
            for w, x, m in zip(want, raw, (d, dv)):
                w[s, h, :len(k), :rb(m)] = x[s, :, h, 16:16 + rb(m)].cpu()[torch.from_numpy(k).long()]
    assert np.array_equal(mo.cpu().numpy(), wm) and np.array_equal(po.cpu().numpy(), wp)
    for w, x in zip(want, out):
        assert torch.equal(x.cpu(), w)


def test_evict_new_outputs_captured_and_refusals():
    S, HK, n, n_keep = 2, 2, 600, 128
    mass, pos = evict_case(S, HK, n, 1)
    past = torch.tensor([2 * n + 3] * S, dtype=torch.int32).cuda()
    m, p = torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda()
    k, v = (torch.randn((S, HK, n, 64), generator=gen(s)).half().cuda() for s in (1, 2))
    used = torch.tensor([n, n], dtype=torch.int32).cuda()
    run = lambda: ops.kv_evict(m, p, past, n_keep, 4, 32, n_used=used, k=k, v=v)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, evicted, mo, po, ko, vo = run()
    for seed, u in ((2, [600, 600]), (3, [600, 50]), (4, [0, 599]), (5, [600, 128])):
        mass, pos = evict_case(S, HK, n, seed)
        m.copy_(torch.from_numpy(mass)); p.copy_(torch.from_numpy(pos)); used.copy_(torch.tensor(u, dtype=torch.int32))
        ko.zero_(); vo.zero_()
        graph.replay()
        torch.cuda.synchronize()
        wk, we = evict_oracle(mass, pos, past.cpu().numpy(), u, n_keep, n - n_keep, 4, 32)
        assert np.array_equal(kept.cpu().numpy(), wk) and np.array_equal(evicted.cpu().numpy(), we)
        for x, y in ((k, ko), (v, vo)):
            for s in range(S):
                for h in range(HK):
                    i = torch.from_numpy(wk[s, h][wk[s, h] >= 0]).long()
                    assert torch.equal(y[s, h, :len(i)].cpu(), x[s, h].cpu()[i]) and (y[s, h, len(i):] == 0).all()
    with pytest.raises(K.Mi355Error):
        ops.kv_evict(m, p, past, 0)
    with pytest.raises(K.Mi355Error):
        ops.kv_evict(m, p, past, 10, 6, 5)
    with pytest.raises(K.Mi355Error):
        ops.kv_evict(m, p, past, n, k=k, v=v, k_out=k, v_out=v)
    for bad in (dict(k=k), dict(k=k, v=v.float()), dict(k=k, v=v, k_out=ko), dict(k=k, v=v[:, :, :5]), dict(n_used=used.long())):
        with pytest.raises(ValueError):
            ops.kv_evict(m, p, past, n_keep, **bad)
    with pytest.raises(ValueError):
        ops.kv_evict(m.double(), p, past, n_keep)
    kept, evicted = ops.kv_evict(m[:, :, :0], p[:, :, :0], past, 3)
    assert (kept == -1).all() and evicted.shape == (S, HK, 0)


@pytest.mark.parametrize("n", [9, 1500, 5000, 20000, 40000])
def test_evict_keeps_sinks_and_recent_slots_before_any_mass(n):
    """a mass of +inf (a sum that overflowed) is the largest mass and no more: it does not take the place of a sink or of a recent position"""
    r = np.random.default_rng(n)
    mass = r.random((1, 2, n)).astype(np.float32)
    mass[:, :, : n - 4] = np.inf
    pos = np.stack([np.arange(n), n - 1 - np.arange(n)])[None].astype(np.int32)          # sinks at the lowest slots, and at the highest
    past = torch.full((1,), n, dtype=torch.int32, device="cuda")
    for n_keep, sink, recent in ((4, 2, 2), (5, 1, 3), (n - 2, 2, 2), (2, 0, 2), (3, 3, 0)):
        kept, evicted = ops.kv_evict(torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda(), past, n_keep, sink, recent)
        for h in range(2):
            pinned = np.nonzero((pos[0, h] < sink) | (pos[0, h] >= n - recent))[0]
            others = [j for j in np.lexsort((np.arange(n), -mass[0, h].astype(np.float64))) if j not in set(pinned)]
            want = np.sort(np.concatenate([pinned, np.array(others[: n_keep - len(pinned)], dtype=np.int64)]))
            assert np.array_equal(kept[0, h].cpu().numpy(), want)
            assert np.array_equal(evicted[0, h].cpu().numpy(), np.setdiff1d(np.arange(n), want))


@pytest.mark.parametrize("t", [B.F16, B.Q8_0])
@pytest.mark.parametrize("S,n", [(0, 10), (2, 0), (0, 0)])
def test_evict_of_no_sequences_or_slots(S, n, t):
    """with and without caches: empty results, -1 and 0 where nothing is kept"""
    HK, n_keep, row = 2, 3, 64 if t in DTYPE else 2 * B.TYPE_SIZE[t]
    mass, pos, past = torch.zeros((S, HK, n), device="cuda"), torch.zeros((S, HK, n), dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")
    kept, evicted = ops.kv_evict(mass, pos, past, n_keep)
    assert kept.shape == (S, HK, n_keep) and (kept == -1).all() and evicted.shape == (S, HK, max(0, n - n_keep))
    k, v = (torch.zeros((S, HK, n, row), dtype=DTYPE.get(t, torch.uint8), device="cuda") for _ in range(2))
    kept, _, mo, po, ko, vo = ops.kv_evict(mass, pos, past, n_keep, 1, 1, n_used=past, k=k, v=v, type_kv=t)
    assert (kept == -1).all() and (mo == 0).all() and (po == -1).all() and ko.shape == vo.shape == (S, HK, n_keep, row) and (ko == 0).all() and (vo == 0).all()


@pytest.mark.parametrize("layout", ["behind", "turns", "side", "halves", "slots"])
def test_evict_gathers_into_the_caches_own_buffer(layout):
    """outputs in the same allocation as the caches, no byte in common: taken, and the caches stay as they were"""
    S, HK, n, n_keep, d = 2, 3, 100, 40, 64
    mass, pos = evict_case(S, HK, n, 5)
    past = torch.full((S,), 2 * n + 3, dtype=torch.int32, device="cuda")
    if layout == "behind":                       # one after the other
        raw = torch.randn((2 * S * HK * (n + n_keep) * d,), generator=gen(1)).half().cuda()
        sizes = [S * HK * m * d for m in (n, n, n_keep, n_keep)]
        k, v, ko, vo = (x.view(S, HK, -1, d) for x in raw.split(sizes))
    elif layout == "turns":                      # every head's slots, then the room for its copy
        raw = torch.randn((2, S, HK, n + n_keep, d), generator=gen(1)).half().cuda()
        (k, v), (ko, vo) = raw[:, :, :, :n], raw[:, :, :, n:]
    elif layout == "side":                       # K and V of a slot side by side, so are their copies
        raw = torch.randn((S, HK, n + n_keep, 2, d), generator=gen(1)).half().cuda()
        k, v, ko, vo = raw[:, :, :n, 0], raw[:, :, :n, 1], raw[:, :, n:, 0], raw[:, :, n:, 1]
    elif layout == "halves":                     # each slot's K, V and two rows of a copy
        raw = torch.randn((S, HK, n, 4, d), generator=gen(1)).half().cuda()
        k, v, ko, vo = raw[:, :, :, 0], raw[:, :, :, 1], raw[:, :, :n_keep, 2], raw[:, :, :n_keep, 3]
    else:                                        # slot-major: all heads of a slot side by side
        raw = torch.randn((S, n + n_keep, 2, HK, d), generator=gen(1)).half().cuda()
        k, v, ko, vo = (x.transpose(1, 2) for x in (raw[:, :n, 0], raw[:, :n, 1], raw[:, n:, 0], raw[:, n:, 1]))
    before = k.clone(), v.clone()
    kept, _, mo, po = ops.kv_evict(torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda(), past, n_keep, 4, 10, k=k, v=v, k_out=ko, v_out=vo)
    wk, _ = evict_oracle(mass, pos, past.cpu().numpy(), [n] * S, n_keep, 0, 4, 10)
    assert np.array_equal(kept.cpu().numpy(), wk) and torch.equal(k, before[0]) and torch.equal(v, before[1])
    at = (torch.arange(S)[:, None, None], torch.arange(HK)[None, :, None], torch.from_numpy(wk).long())
    assert torch.equal(ko.cpu(), before[0].cpu()[at]) and torch.equal(vo.cpu(), before[1].cpu()[at])
    with pytest.raises(K.Mi355Error):            # a shifted view of the cache itself
        ops.kv_evict(torch.from_numpy(mass).cuda(), torch.from_numpy(pos).cuda(), past, n_keep, 4, 10, k=k, v=v, k_out=k[:, :, 1:1 + n_keep], v_out=vo)


# ---- attention with the weight every slot draws ----------------------------------------------------------------------------------------

def attn_oracle(q, k, v, mask, scale, mass, decay, max_bias=0.0, softcap=0.0):
    """f64 on the CPU: (dst [S, n, H, dv] | None, its bound, mass, its bound).  q [S, H, n, d], k / v f64 values, mask f16 [1 | S, 1 | H, >= n, slots]"""
    S, H, n, d = q.shape
    HK, slots = k.shape[1], k.shape[2]
    G = H // HK
    kk = k.repeat_interleave(G, 1)
    hidden = torch.zeros((1, 1, 1, slots), dtype=torch.bool) if mask is None else mask[:, :, :n].double() == float("-inf")
    m = torch.zeros((1, 1, 1, slots), dtype=torch.float64) if mask is None else torch.where(hidden, 0.0, mask[:, :, :n].double())
    if max_bias > 0:
        p2 = 1 << int(math.floor(math.log2(H)))
        m0, m1 = 2.0 ** (-max_bias / p2), 2.0 ** (-max_bias / 2 / p2)
        sl = torch.tensor([m0 ** (h + 1) if h < p2 else m1 ** (2 * (h - p2) + 1) for h in range(H)], dtype=torch.float64)
        m = m * sl[None, :, None, None]
    qd = q.double()
    ok = (~hidden).expand(S, H, n, slots)
    # slots that no query sees may hold anything
    seen = ok.any(1).any(1)[:, None, :, None] if mask is not None else None
    clean = lambda x: x if seen is None else torch.where(seen, x, torch.zeros((), dtype=torch.float64))  # noqa: E731
    kk = clean(kk)
    dot, mag = qd @ kk.transpose(2, 3), qd.abs() @ kk.abs().transpose(2, 3)
    s = softcap * torch.tanh(dot * scale / softcap) if softcap else dot * scale
    s = s + m
    # a logit: products and sum of d terms in any order, scale, mask; tanh to 8 steps
    es = (d + 10) * U32 * abs(scale) * mag + 6 * U32 * (s.abs() + m.abs()) + (8 * U32 * abs(softcap))
    es = torch.where(ok, es, torch.zeros((), dtype=torch.float64)).amax(-1, keepdim=True)
    s = torch.where(ok, s, torch.full((), float("-inf"), dtype=torch.float64))
    top = s.amax(-1, keepdim=True)
    p = torch.where(ok, torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top)), torch.zeros((), dtype=torch.float64))
    tot = p.sum(-1, keepdim=True)
    p = torch.where(tot > 0, p / tot, torch.zeros((), dtype=torch.float64))
    # p: its logit and those of the sum, exp and its argument (|s - top| in steps of 2^-24), the sum of the slots in any order
    span = torch.where(ok, (s - top).abs(), torch.zeros((), dtype=torch.float64))
    span = torch.where(p > 1e-12, span, torch.zeros_like(span)).amax(-1, keepdim=True)
    rel = 2 * es + (10 + slots + 4 * span) * U32
    w = (p * (1 + 0 * rel)).reshape(S, HK, G * n, slots)
    wm = w.sum(2) + (decay * mass.double() if mass is not None and decay != 0 else 0.0)
    em = (p * rel).reshape(S, HK, G * n, slots).sum(2) + (G * n + 4) * U32 * wm.abs() + G * n * 2.0 ** -126
    if v is None:
        return None, None, wm, em
    vv = clean(v.repeat_interleave(G, 1))
    o = (p @ vv).transpose(1, 2)
    eo = (((p * rel) @ vv.abs()) + (slots + 4) * U32 * (p @ vv.abs())).transpose(1, 2) + 2.0 ** -126
    return o, eo, wm, em


def check_attn(q, kc, vc, t, mask, scale, mass, decay, near=True, **kw):
    """through both entry points (vc None: attn_mass alone)"""
    dev = lambda x: x.cuda() if x is not None else None  # noqa: E731
    k64, v64 = values(kc, t), values(vc, t) if vc is not None else None
    wd, ed, wm, em = attn_oracle(q, k64, v64, mask[None, None] if mask is not None and mask.dim() == 2 else mask, scale, mass, decay, **kw)
    o = dict(max_bias=kw.get("max_bias", 0.0), logit_softcap=kw.get("softcap", 0.0))
    got = ops.attn_mass(dev(q), dev(kc), dev(mask), t, scale, mass=dev(mass), decay=decay, **o).cpu().double()
    assert ((got - wm).abs() <= em).all(), float(((got - wm).abs() / em).max())
    if vc is not None:
        d1, m1 = ops.flash_attn_ext_mass(dev(q), dev(kc), dev(vc), dev(mask), t, scale, mass=dev(mass), decay=decay, **o)
        d1, m1 = d1.cpu().double(), m1.cpu().double()
        assert ((m1 - wm).abs() <= em).all(), float(((m1 - wm).abs() / em).max())
        assert ((d1 - wd).abs() <= ed).all(), float(((d1 - wd).abs() / ed).max())
        if near and wd.norm() > 0:       # roundings of random inputs do not add up: far below the bounds above, which hold for any input
            assert (d1 - wd).norm() <= 1e-5 * wd.norm()
    if near and wm.norm() > 0:
        assert (got - wm).norm() <= 1e-5 * wm.norm()


def attn_case(S, H, HK, n, slots, d, dv, t, seed, qscale=1.5):
    g = gen(seed)
    return (torch.randn((S, H, n, d), generator=g) * qscale, cache((S, HK, slots, d), t, g), cache((S, HK, slots, dv), t, g) if dv else None,
            torch.rand((S, HK, slots), generator=g) * 2)


def causal(S, n, slots, lens=None, pad=0):
    lens = lens or [slots] * S
    j, i = torch.arange(slots), torch.arange(n + pad)
    m = torch.stack([torch.where(j[None] < torch.clamp(torch.tensor(L) - (n - 1 - i[:, None]), min=0), 0.0, float("-inf")) for L in lens])
    return m.half()[:, None]


ATTN = [
    # S, H, HK, n, slots, d, dv, type
    (1, 32, 8, 1, 512, 128, 128, B.F16), (1, 8, 8, 1, 1, 64, 64, B.F16), (1, 8, 2, 1, 2, 128, 128, B.Q8_0), (2, 4, 1, 2, 63, 64, 64, B.BF16),
    (1, 16, 2, 3, 65, 128, 128, B.Q4_0), (3, 6, 2, 1, 257, 96, 64, B.F16), (1, 12, 1, 8, 130, 128, 128, B.F16), (2, 5, 5, 4, 300, 80, 80, B.F16),
    (1, 8, 1, 5, 1000, 256, 256, B.F16), (1, 8, 1, 5, 1000, 256, 128, B.BF16), (1, 32, 8, 8, 777, 128, 128, B.Q8_0), (1, 64, 8, 1, 4099, 128, 128, B.F16),
    (2, 32, 8, 1, 3000, 128, 128, B.Q4_0), (1, 2, 1, 1, 40, 8, 8, B.F16), (1, 32, 1, 8, 200, 64, 64, B.Q8_0), (1, 3, 1, 7, 129, 72, 40, B.BF16),
    (4, 8, 4, 1, 1500, 32, 32, B.Q4_0), (1, 40, 8, 6, 520, 112, 112, B.F16), (1, 64, 1, 1, 333, 192, 128, B.F16), (9, 4, 2, 1, 31, 160, 96, B.Q8_0),
]


@pytest.mark.parametrize("S,H,HK,n,slots,d,dv,t", ATTN)
def test_attention_mass_of_a_step(S, H, HK, n, slots, d, dv, t):
    q, k, v, mass = attn_case(S, H, HK, n, slots, d, dv, t, slots + d)
    lens = [max(n, slots - i * slots // (2 * S)) for i in range(S)]
    check_attn(q, k, v, t, causal(S, n, slots, [min(L, slots) for L in lens], pad=3), 1 / math.sqrt(d), mass, 0.9)


@pytest.mark.parametrize("S,H,HK,n,slots,d,t", [
    (1, 8, 2, 17, 33, 64, B.F16), (1, 32, 8, 64, 1000, 128, B.F16), (2, 4, 1, 33, 300, 128, B.Q8_0), (1, 6, 2, 100, 100, 96, B.BF16), (1, 4, 4, 257, 257, 64, B.Q4_0),
    (1, 5, 1, 70, 515, 256, B.F16), (1, 2, 2, 9, 2049, 80, B.F16), (3, 8, 8, 12, 140, 128, B.BF16), (1, 64, 8, 10, 130, 128, B.Q4_0), (1, 4, 2, 300, 900, 128, B.F16),
    (1, 8, 1, 520, 520, 128, B.BF16), (1, 1, 1, 1, 5000, 128, B.Q8_0), (1, 3, 1, 130, 65, 8, B.F16),
    (8, 64, 64, 9, 300, 64, B.F16), (1, 4, 2, 20, 1, 128, B.F16), (1, 4, 1, 9, 31, 64, B.Q8_0), (2, 2, 1, 64, 64, 128, B.BF16), (1, 8, 8, 33, 257, 128, B.Q4_0), (1, 7, 1, 37, 511, 192, B.BF16),
])
def test_attention_mass_of_a_prompt(S, H, HK, n, slots, d, t):
    q, k, _, mass = attn_case(S, H, HK, n, slots, d, 0, t, slots + n)
    check_attn(q, k, None, t, causal(S, n, slots), 1 / math.sqrt(d), mass, 1.0)
    check_attn(q, k, None, t, None, 1 / math.sqrt(d), None, 1.0)


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_mass_of_prompts_that_fill_the_card(t, d):
    """so many heads that a workgroup has many tiles of slots and of rows: they go round the places in LDS several times"""
    S, H, HK, n, slots = 2, 32, 16, 200, 1000
    q, k, _, mass = attn_case(S, H, HK, n, slots, d, 0, t, d)
    check_attn(q, k, None, t, causal(S, n, slots, [slots, 700]), 1 / math.sqrt(d), mass, 1.0)


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attention_mass_masks(t, n):
    """queries that see nothing, masks per head, biases, the lowest value in every place; hidden rows of NaN and infinities"""
    S, H, HK, slots, d = 2, 8, 2, 200, 128
    q, k, v, mass = attn_case(S, H, HK, n, slots, d, d if n <= 8 else 0, t, n)
    g = gen(n)
    mask = torch.where(torch.rand((S, H, n, slots), generator=g) < 0.3, float("-inf"), 0.0) + torch.randn((S, H, n, slots), generator=g)
    mask[0, 1, 0], mask[1, :, n - 1], mask[0, 5, :, 7] = float("-inf"), float("-inf"), float("-inf")
    mask[..., 100:140] = float("-inf")                        # hidden from everyone
    mask[0, 3, 0, 1:] = float("-inf")                         # one slot left
    mask = mask.half()
    for bad in ((k, v) if v is not None else (k,)):
        if t in DTYPE:
            bad[:, :, 100:120], bad[:, :, 120:130], bad[:, :, 130:140] = float("nan"), float("inf"), float("-inf")
        else:
            bad[:, :, 100:140] = 255                           # a scale of NaN
    check_attn(q, k, v, t, mask, 1 / math.sqrt(d), mass, 0.5)
    check_attn(q, k, v, t, mask, 1 / math.sqrt(d), mass, 0.5, max_bias=8.0)
    low = torch.full((1, 1, n, slots), -65504.0).half()
    low[..., 100:140] = float("-inf")
    check_attn(q, k, v, t, low, 1 / math.sqrt(d), mass, 0.5, near=False)
    low[..., 50] = 0.0                                        # one slot beside the lowest values: it draws everything
    check_attn(q, k, v, t, low, 1 / math.sqrt(d), mass, 0.5, near=False)


@pytest.mark.parametrize("t", [B.F16, B.Q8_0])
def test_attention_mass_hidden_from_one_head_only(t):
    """a row of NaN that one head sees spoils that head's result and no other's"""
    H, HK, slots, d, n = 4, 2, 70, 64, 2
    q, k, v, mass = attn_case(1, H, HK, n, slots, d, d, t, 3)
    mask = torch.zeros((1, H, n, slots)).half()
    mask[0, [0, 2, 3], :, 9] = float("-inf")
    for x in (k, v):
        if t in DTYPE:
            x[:, :, 9] = float("nan")
        else:
            x[:, :, 9] = 255
    dst, _ = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), mask.cuda(), t, 0.125)
    assert torch.isnan(dst[0, :, 1]).all() and torch.isfinite(dst[0, :, [0, 2, 3]]).all()


@pytest.mark.parametrize("n", [1, 3, 50])
def test_attention_mass_softcap_bias_and_sharp_logits(n):
    S, H, HK, slots, d = 1, 6, 2, 333, 128
    q, k, v, mass = attn_case(S, H, HK, n, slots, d, d if n <= 8 else 0, B.F16, 40 + n)
    check_attn(q, k, v, B.F16, causal(S, n, slots), 0.088, mass, 1.0, softcap=30.0)
    check_attn(q * 20, k, v, B.F16, causal(S, n, slots), 0.088, mass, 1.0, near=False)                 # almost all weight on single slots
    check_attn(q * 1e-3, k, v, B.F16, None, 0.088, mass, 1.0)                                        # almost equal weights
    big = q.clone()
    big[..., 0] *= 1e6                                                                               # beyond the range of f16
    check_attn(big, k, v, B.F16, causal(S, n, slots), 1e-6, mass, 1.0, near=False)


def test_attention_mass_strided_caches_in_place_and_unread():
    """slot-major caches (every head's rows of a slot side by side), q as [seq, token, head, d], mass_out on mass, decay 0 over NaN"""
    S, H, HK, n, slots, d = 2, 8, 2, 2, 150, 128
    for t in (B.F16, B.Q8_0, B.Q4_0):
        g = gen(t)
        q = torch.randn((S, n, H, d), generator=g)
        k, v = (cache((S, slots, HK, d), t, g) for _ in range(2))
        mass = torch.rand((S, HK, slots + 5), generator=g)
        mask = causal(S, n, slots)
        kg, vg, qg, mg = k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), q.cuda().transpose(1, 2), mass.cuda()
        wd, ed, wm, em = attn_oracle(q.transpose(1, 2), values(k.transpose(1, 2), t), values(v.transpose(1, 2), t), mask, 0.1, mass[..., :slots], 0.75)
        dst, out = ops.flash_attn_ext_mass(qg, kg, vg, mask.cuda(), t, 0.1, mass=mg[..., :slots], decay=0.75, mass_out=mg[..., :slots])
        assert out.data_ptr() == mg.data_ptr() and ((dst.cpu().double() - wd).abs() <= ed).all() and ((mg[..., :slots].cpu().double() - wm).abs() <= em).all()
        assert torch.equal(mg[..., slots:].cpu(), mass[..., slots:])
        _, _, wm, em = attn_oracle(q.transpose(1, 2), values(k.transpose(1, 2), t), None, mask, 0.1, None, 0.0)
        nan = torch.full((S, HK, slots), float("nan"), device="cuda")
        for got in (ops.flash_attn_ext_mass(qg, kg, vg, mask.cuda(), t, 0.1, mass=nan, decay=0.0)[1], ops.attn_mass(qg, kg, mask.cuda(), t, 0.1, mass=nan, decay=0.0)):
            assert ((got.cpu().double() - wm).abs() <= em).all()


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("n", [1, 8, 20])
def test_attention_mass_is_as_exact_as_f32(t, n):
    """the operands are split into 16-bit parts: no further from 64 bits than the same sums in f32 torch, in dst and in the weights"""
    S, H, HK, slots, d = 1, 16, 4, 2500, 128
    q, k, v, _ = attn_case(S, H, HK, n, slots, d, d, t, 90 + n)
    mask = causal(S, n, slots)
    k64, v64 = values(k, t), values(v, t)
    wd, _, wm, _ = attn_oracle(q, k64, v64, mask, 0.09, None, 0.0)
    s = (q @ k64.float().repeat_interleave(4, 1).transpose(2, 3)) * 0.09 + mask.float()
    p = torch.softmax(s, -1)
    fd, fm = (p @ v64.float().repeat_interleave(4, 1)).transpose(1, 2), p.reshape(S, HK, 4 * n, slots).sum(2)
    far = lambda x, y: float((x.cpu().double() - y).norm() / y.norm())  # noqa: E731
    if n <= 8:
        dst, mass = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), mask.cuda(), t, 0.09)
        assert far(dst, wd) <= 1.5 * far(fd, wd) + 3e-7
    else:
        mass = ops.attn_mass(q.cuda(), k.cuda(), mask.cuda(), t, 0.09)
    assert far(mass, wm) <= 1.5 * far(fm, wm) + 3e-7


@pytest.mark.parametrize("n", [1, 24])
def test_attention_mass_offsets_past_32_bits(n):
    """slots 100 MiB apart: the last rows lie beyond 4 GiB"""
    H, HK, slots, d, step = 4, 1, 48, 128, 100 << 20
    q, k, v, mass = attn_case(1, H, HK, n, slots, d, d, B.F16, 77)
    raw = torch.empty(step * slots, dtype=torch.uint8, device="cuda")
    far = lambda off: raw.view(torch.float16).as_strided((1, HK, slots, d), (0, 0, step // 2, 1), off)  # noqa: E731
    kg, vg = far(0), far(4096)
    kg.copy_(k), vg.copy_(v)
    mask = causal(1, n, slots)
    wd, ed, wm, em = attn_oracle(q, values(k, B.F16), values(v, B.F16), mask, 0.1, mass, 1.0)
    assert ((ops.attn_mass(q.cuda(), kg, mask.cuda(), B.F16, 0.1, mass=mass.cuda()).cpu().double() - wm).abs() <= em).all()
    if n <= 8:
        dst, out = ops.flash_attn_ext_mass(q.cuda(), kg, vg, mask.cuda(), B.F16, 0.1, mass=mass.cuda())
        assert ((dst.cpu().double() - wd).abs() <= ed).all() and ((out.cpu().double() - wm).abs() <= em).all()


def test_attention_mass_two_streams_captured_and_nothing_cached():
    """two captured graphs with workspaces of their own, replayed on two streams at once, inputs changed between the replays; an empty cache"""
    S, H, HK, slots, d = 1, 32, 8, 3000, 128
    sides = [torch.cuda.Stream() for _ in range(2)]
    state = []
    for i, n in enumerate((1, 30)):
        q, k, v, mass = attn_case(S, H, HK, n, slots, d, d, B.F16, i)
        dev = [x.cuda() for x in (q, k, v, mass, causal(S, n, slots))]
        out = torch.empty((S, HK, slots), device="cuda")
        def run(dev=dev, n=n, out=out):
            q, k, v, mass, mask = dev
            if n <= 8:
                return ops.flash_attn_ext_mass(q, k, v, mask, B.F16, 0.09, mass=mass, mass_out=out)
            return ops.attn_mass(q, k, mask, B.F16, 0.09, mass=mass, mass_out=out)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        state.append((graph, dev, res, run, out))
    for rep in range(4):
        for graph, dev, *_ in state:
            dev[0].copy_(torch.randn(dev[0].shape, generator=gen(50 + rep)))
            dev[3].copy_(torch.rand(dev[3].shape, generator=gen(60 + rep)))
        torch.cuda.synchronize()
        for side, (graph, *_) in zip(sides, state):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, dev, res, run, out in state:
            got = [x.clone() for x in (res if isinstance(res, tuple) else (res,))]
            want = run()
            for x, y in zip(got, want if isinstance(want, tuple) else (want,)):
                assert torch.equal(x, y)          # no atomics: the same bits every time
    q = torch.randn((1, 4, 1, 64), device="cuda")
    none = torch.zeros((1, 2, 0, 64), dtype=torch.float16, device="cuda")
    dst, mass = ops.flash_attn_ext_mass(q, none, none, None, B.F16, 0.1)
    assert (dst == 0).all() and mass.shape == (1, 2, 0)


def test_attention_mass_wrapper_refuses_what_does_not_fit():
    q, k, v, mass = (x.cuda() for x in attn_case(1, 4, 2, 1, 10, 64, 64, B.F16, 1))
    ok = dict(q=q, k=k, v=v, mask=None, type_kv=B.F16, scale=0.1)
    for bad in (dict(q=q.half()), dict(k=k.float()), dict(k=k[..., :32]), dict(v=v[:, :, :5]), dict(mask=torch.zeros((1, 5), device="cuda").half()),
                dict(mask=torch.zeros((1, 10), device="cuda")), dict(mass=mass.double()), dict(mass_out=mass[:, :, :3]), dict(type_kv=B.Q8_0), dict(k=k.cpu())):
        with pytest.raises(ValueError):
            ops.flash_attn_ext_mass(**{**ok, **bad})
    with pytest.raises(K.Mi355Error):
        ops.flash_attn_ext_mass(q.expand(1, 4, 9, 64).contiguous(), k, v, None, B.F16, 0.1)
    with pytest.raises(K.Mi355Error):
        ops.flash_attn_ext_mass(q[:, :3], k, v, None, B.F16, 0.1)


def test_attention_mass_takes_a_mask_of_f16_or_its_bits_only():
    """another 16-bit type's bits would be read as f16: bf16's -inf is a NaN there"""
    q, k, v, _ = (x.cuda() for x in attn_case(1, 4, 2, 1, 40, 64, 64, B.F16, 1))
    mask = causal(1, 1, 40, [30]).cuda()
    want = ops.flash_attn_ext_mass(q, k, v, mask, B.F16, 0.1)
    for same in (mask.view(torch.int16), mask.view(torch.uint16)):
        got = ops.flash_attn_ext_mass(q, k, v, same, B.F16, 0.1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(ops.attn_mass(q, k, same, B.F16, 0.1), ops.attn_mass(q, k, mask, B.F16, 0.1))
    for bad in (mask.bfloat16(), mask.float(), mask == 0, mask.double()):
        with pytest.raises(ValueError):
            ops.flash_attn_ext_mass(q, k, v, bad, B.F16, 0.1)
        with pytest.raises(ValueError):
            ops.attn_mass(q, k, bad, B.F16, 0.1)


def test_attention_mass_refuses_a_mask_of_other_sequences_or_heads():
    """planes that neither are one nor go into the sequences or heads evenly would be dealt out in turn"""
    q, k, v, _ = (x.cuda() for x in attn_case(2, 6, 2, 1, 40, 64, 64, B.F16, 1))
    for shape in ((3, 1, 1, 40), (1, 4, 1, 40), (2, 12, 1, 40), (4, 1, 1, 40), (3, 1, 40), (0, 1, 1, 40), (1, 0, 1, 40)):
        with pytest.raises(ValueError):
            ops.flash_attn_ext_mass(q, k, v, torch.zeros(shape, device="cuda").half(), B.F16, 0.1)
        with pytest.raises(ValueError):
            ops.attn_mass(q, k, torch.zeros(shape, device="cuda").half(), B.F16, 0.1)


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("n", [1, 8, 40])
@pytest.mark.parametrize("cap", [30.0, 50.0, 1000.0])
def test_attention_mass_softcap_is_exact_relative_to_the_logit(t, n, cap):
    """one feature of q is not zero, so a logit is one product and what is left of its error is the cap's: a few steps of the logit itself,
    whatever the cap"""
    H, HK, slots, d, scale = 8, 2, 40, 128, 0.125
    g = gen(int(cap) + n)
    q = torch.zeros((1, H, n, d))
    q[..., 32] = torch.randn((1, H, n), generator=g) * 16
    k = cache((1, HK, slots, d), t, g)
    dot = q.double() @ values(k, t).repeat_interleave(H // HK, 1).transpose(2, 3)
    s = cap * torch.tanh(dot * scale / cap)
    # q in parts (4 steps of 2^-24), the parts' products and the block's scale (3), scale / cap, its product, the row's power of two (3), tanh (8), cap (2);
    # the weight: its logit and those of the sum, exp and its argument, the sum over the slots
    es = (20 * U32 * s.abs()).amax(-1, keepdim=True)
    span = (s - s.amax(-1, keepdim=True)).abs().amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    rel = 2 * es + (10 + slots + 4 * span) * U32
    fold = lambda x: x.reshape(1, HK, -1, slots).sum(2)  # noqa: E731
    want, err = fold(p), fold(p * rel) + (H // HK * n + 4) * U32 * fold(p)
    assert ((ops.attn_mass(q.cuda(), k.cuda(), None, t, scale, logit_softcap=cap).cpu().double() - want).abs() <= err).all()
    if n <= 8:
        v = cache((1, HK, slots, d), t, g)
        dst, mass = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), None, t, scale, logit_softcap=cap)
        assert ((mass.cpu().double() - want).abs() <= err).all()
        vv = values(v, t).repeat_interleave(H // HK, 1)
        bound = (p * rel) @ vv.abs() + (slots + 4) * U32 * (p @ vv.abs())
        assert ((dst.cpu().double() - (p @ vv).transpose(1, 2)).abs() <= bound.transpose(1, 2) + 2.0 ** -126).all()


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("cap", [30.0, 50.0, 1000.0])
def test_attention_mass_softcap_is_as_exact_as_f32(t, n, cap):
    """no further from 64 bits than the same formula in f32 torch"""
    H, HK, slots, d = 16, 4, 700, 128
    q, k, _, _ = attn_case(1, H, HK, n, slots, d, 0, t, 7 + n)
    kk = values(k, t).repeat_interleave(H // HK, 1).transpose(2, 3)
    fold = lambda s: torch.softmax(s, -1).reshape(1, HK, -1, slots).sum(2)  # noqa: E731
    want = fold(cap * torch.tanh(q.double() @ kk * 0.09 / cap))
    f32 = fold(cap * torch.tanh((q @ kk.float()) * 0.09 / cap))
    got = ops.attn_mass(q.cuda(), k.cuda(), None, t, 0.09, logit_softcap=cap)
    far = lambda x: float((x.cpu().double() - want).norm() / want.norm())  # noqa: E731
    assert far(got) <= 1.5 * far(f32) + 3e-7


@pytest.mark.parametrize("t", [B.F16, B.BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attention_mass_of_keys_with_infinities(t, d, n):
    """a logit of -inf is a weight of 0, as if the slot were hidden; one of +inf makes its own query's results NaN and no other's"""
    H, HK, slots, scale = 8, 2, 300, 0.08
    q, k, v, _ = attn_case(1, H, HK, n, slots, d, d, t, d + n)
    q[..., 7], q[..., 40] = -q[..., 7].abs() - 0.1, q[..., 40].abs() * 1e-3 + 1e-4
    out = [3, 31, 32, 100, 201, 299]
    k[:, :, out[::2], 7], k[:, :, out[1::2], 40] = float("inf"), float("-inf")
    mask = causal(1, n, slots)
    hidden, clean = mask.clone(), k.clone()
    hidden[..., out] = float("-inf")
    clean[:, :, out] = 0.0
    wd, ed, wm, em = attn_oracle(q, values(clean, t), values(v, t), hidden, scale, None, 0.0)
    args = (k.cuda(), mask.cuda(), t, scale)
    assert ((ops.attn_mass(q.cuda(), *args).cpu().double() - wm).abs() <= em).all()
    if n <= 8:
        dst, mass = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), mask.cuda(), t, scale)
        assert ((dst.cpu().double() - wd).abs() <= ed).all() and ((mass.cpu().double() - wm).abs() <= em).all()
    q[0, 5, n - 1, 7] = 1.0                                   # the other sign: +inf among the logits of head 5's last query
    mass = ops.attn_mass(q.cuda(), *args).cpu()
    _, _, wm, em = attn_oracle(q[:, :4], values(clean, t)[:, :1], None, hidden, scale, None, 0.0)
    assert torch.isnan(mass[0, 1, out[0]]) and ((mass[:, :1].double() - wm).abs() <= em).all()
    if n <= 8:
        dst, _ = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), args[1], t, scale)
        other = torch.ones((n, H), dtype=torch.bool)
        other[n - 1, 5] = False
        assert torch.isnan(dst[0, n - 1, 5]).all() and ((dst.cpu().double() - wd).abs() <= ed)[0][other].all()


@pytest.mark.parametrize("t", [B.F16, B.BF16])
@pytest.mark.parametrize("d", [8, 72, 80, 96, 112, 160, 192, 248])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_attention_mass_of_infinities_at_the_end_of_a_key(t, d, n):
    """heads that a larger size's kernel serves: what it reads in place of the features past the head size does not count"""
    H, HK, slots, scale = 4, 2, 90, 0.1
    q, k, v, _ = attn_case(1, H, HK, n, slots, d, d, t, d + n)
    q[..., d - 1] = -q[..., d - 1].abs() - 0.1
    out = [0, 5, 40, 64, 89]
    k[:, :, out, d - 1] = float("inf")
    hidden, clean = torch.zeros((1, 1, n, slots)).half(), k.clone()
    hidden[..., out], clean[:, :, out] = float("-inf"), 0.0
    wd, ed, wm, em = attn_oracle(q, values(clean, t), values(v, t), hidden, scale, None, 0.0)
    assert ((ops.attn_mass(q.cuda(), k.cuda(), None, t, scale).cpu().double() - wm).abs() <= em).all()
    if n <= 8:
        dst, mass = ops.flash_attn_ext_mass(q.cuda(), k.cuda(), v.cuda(), None, t, scale)
        assert ((dst.cpu().double() - wd).abs() <= ed).all() and ((mass.cpu().double() - wm).abs() <= em).all()


@pytest.mark.parametrize("S,n,slots", [(1, 0, 5), (2, 0, 512), (1, 0, 100000), (0, 1, 512), (0, 40, 300), (1, 0, 0)])
def test_attention_mass_of_no_queries(S, n, slots):
    """an empty batch: an empty dst, and what earlier calls left, decayed"""
    q = torch.zeros((S, 8, n, 64), device="cuda")
    k = torch.zeros((S, 2, slots, 64), dtype=torch.float16, device="cuda")
    mass = torch.rand((S, 2, slots), device="cuda")
    for m, decay, want in ((mass, 0.5, mass * 0.5), (None, 1.0, mass * 0), (mass * float("nan"), 0.0, mass * 0)):
        assert torch.equal(ops.attn_mass(q, k, None, B.F16, 0.1, mass=m, decay=decay), want)
        if n <= 8:
            dst, out = ops.flash_attn_ext_mass(q, k, k, None, B.F16, 0.1, mass=m, decay=decay)
            assert dst.shape == (S, n, 8, 64) and torch.equal(out, want)
    got = mass.clone()
    assert ops.attn_mass(q, k, None, B.F16, 0.1, mass=got, decay=0.25, mass_out=got) is got and torch.equal(got, mass * 0.25)


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("n", [2, 40])
def test_attention_mass_hidden_rows_may_be_huge(t, n):
    """rows that no query sees, finite and near the end of the type's range, between rows that all see; visible rows of very different sizes"""
    S, H, HK, slots, d = 1, 4, 2, 300, 128
    q, k, v, mass = attn_case(S, H, HK, n, slots, d, d if n <= 8 else 0, t, 500 + n)
    mask = torch.zeros((1, 1, n, slots)).half()
    mask[..., 3::5] = float("-inf")
    for x in ((k, v) if v is not None else (k,)):
        if t in DTYPE:
            x[:, :, 3::5] = torch.finfo(DTYPE[t]).max / 2 if t == B.F16 else 1e30
            x[:, :, 4::5] *= 2.0 ** -9
        else:
            b = x.view(S, HK, slots, -1, B.TYPE_SIZE[t])
            b[:, :, 3::5, :, :2] = torch.tensor([60000.0]).half().view(torch.uint8)
            b[:, :, 4::5, :, 1] = 0                           # the scale's upper byte: a subnormal one
    check_attn(q, k, v, t, mask, 1 / math.sqrt(d), mass, 0.5)


@pytest.mark.parametrize("t", [B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("G,n,d", [(4, 1, 64), (8, 1, 64), (2, 8, 64), (3, 1, 128), (7, 1, 128), (4, 5, 128), (4, 1, 256), (5, 4, 256), (4, 3, 96), (9, 4, 128)])
def test_attention_mass_of_blocks_at_every_alignment(t, G, n, d):
    """rows that start 2, 4, 8 bytes past 16 and lie an odd number of 2-byte units apart: every way to load them gives the same"""
    HK, slots, size = 2, 203, B.TYPE_SIZE[t] * d // 32
    q, k, v, _ = attn_case(1, G * HK, HK, n, slots, d, d, t, d + G)
    res = []
    for off, pitch in ((0, (size + 15) // 16 * 16), (0, size), (2, size + 2), (4, size + 6), (8, (size + 15) // 16 * 16)):
        def place(x):
            raw = torch.full((HK * slots * pitch + 64,), 255, dtype=torch.uint8, device="cuda")
            y = raw[off:].as_strided((1, HK, slots, size), (0, slots * pitch, pitch, 1), off)
            y.copy_(x)
            return y
        kg, vg = place(k), place(v)
        dst, mass = ops.flash_attn_ext_mass(q.cuda(), kg, vg, None, t, 0.1)
        res.append((dst, mass, ops.attn_mass(q.cuda(), kg, None, t, 0.1)))
    wd, ed, wm, em = attn_oracle(q, values(k, t), values(v, t), None, 0.1, None, 0.0)
    for dst, mass, alone in res:
        assert ((dst.cpu().double() - wd).abs() <= ed).all() and ((mass.cpu().double() - wm).abs() <= em).all() and ((alone.cpu().double() - wm).abs() <= em).all()
        assert torch.equal(dst, res[0][0]) and torch.equal(mass, res[0][1])


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_attention_mass_of_a_prompt_over_strided_caches(t, d):
    """slot-major caches whose rows lie an odd number of the smallest allowed units apart, q as [token, head, d], a mask of odd pitch per sequence"""
    S, H, HK, n, slots = 2, 6, 2, 21, 201
    k, q = cache((S, HK, slots, d), t, gen(d)), torch.randn((S, n, H, d), generator=gen(d + 1))
    width, unit = (k.shape[-1], 8) if t in DTYPE else (k.shape[-1], 2)          # values of 16 bits in 16-byte steps, bytes in 2-byte steps
    off, pitch = 3 * unit, (HK * width + unit + 2 * unit - 1) // (2 * unit) * 2 * unit + unit
    raw = torch.full((S * slots * pitch + off + 64,), 255, dtype=torch.uint8, device="cuda") if t not in DTYPE else torch.full((S * slots * pitch + off + 64,), float("nan"), dtype=k.dtype, device="cuda")
    kg = raw.as_strided((S, HK, slots, width), (slots * pitch, width, pitch, 1), off)
    kg.copy_(k)
    mask = causal(S, n, slots, [slots, 100])
    wide = torch.full((S, 1, n, slots + 6), float("-inf")).half().cuda()
    wide[..., :slots] = mask.cuda()
    _, _, wm, em = attn_oracle(q.transpose(1, 2), values(k, t), None, mask, 0.1, None, 0.0)
    got = ops.attn_mass(q.cuda().transpose(1, 2), kg, wide[..., :slots], t, 0.1)
    assert ((got.cpu().double() - wm).abs() <= em).all()


@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0, B.Q4_0])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_mass_around_one_tile_a_wave(t, d):
    """up to where one launch does it all and one slot beyond, with a full row tile and one row more"""
    for slots in (31, 32, 33, 127, 128, 129, 255, 256, 257):
        for H, HK, n in ((4, 4, 1), (16, 2, 2), (17, 1, 1)):
            q, k, v, mass = attn_case(1, H, HK, n, slots, d, d, t, slots + H)
            check_attn(q, k, v, t, causal(1, n, slots), 1 / math.sqrt(d), mass, 0.9)


@pytest.mark.parametrize("t,d", [(B.Q4_0, 128), (B.F16, 64)])
def test_attention_mass_of_a_long_cache(t, d):
    """more slots than every slice takes in one go; and few queries of a prompt over them"""
    q, k, v, mass = attn_case(1, 4, 2, 1, 140001, d, d, t, 9)
    check_attn(q, k, v, t, None, 1 / math.sqrt(d), mass, 0.9)
    q9 = torch.randn((1, 4, 9, d), generator=gen(1))
    check_attn(q9, k, None, t, causal(1, 9, 140001), 1 / math.sqrt(d), mass, 0.9)


# ---- the operators as they are used --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", [B.F16, B.BF16, B.Q8_0])
def test_prompt_then_decode_in_a_cache_that_stays_full(t):
    """a prompt is stored, its last queries weigh it, its heaviest slots move to the bounded cache; then steps: a token goes to the slot that the
    step before gave up, attention adds up the weights, the next slot is chosen.  The same steps eager and as replays of one graph"""
    S, H, HK, d, n, W, budget, steps = 2, 8, 2, 64, 100, 16, 33, 24
    g = gen(21)
    total = n + steps
    qx, kx, vx = torch.randn((S, total, H, d), generator=g), torch.randn((S, total, HK, d), generator=g), torch.randn((S, total, HK, d), generator=g)
    qw, kw = 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)
    pos = torch.arange(total, dtype=torch.int32)[None].expand(S, total).contiguous()
    qg, kg, vg, pg, qwg, kwg = (x.cuda() for x in (qx, kx, vx, pos, qw, kw))
    scale, opt = 1 / math.sqrt(d), dict(freq_base=10000.0)
    width = d if t in DTYPE else d // 32 * B.TYPE_SIZE[t]
    fresh = lambda slots: torch.zeros((S, HK, slots, width), dtype=DTYPE.get(t, torch.uint8), device="cuda")  # noqa: E731

    # what the cache holds of every token: the operators' own rows, checked once against the formula
    all_k, all_v = fresh(total), fresh(total)
    q_rot = ops.qk_norm_rope(qg, kg, vg, qwg, kwg, 1e-6, pg, all_k, all_v, t, **opt)
    wq, eq = store_oracle(qx, qw, 1e-6, pos, d, 2)
    assert ((q_rot.cpu().double() - wq).abs() <= eq).all()
    if t in DTYPE:
        check_rows(all_k.cpu(), fresh(total).cpu(), torch.arange(total, dtype=torch.int32)[None, None].expand(S, HK, total), *store_oracle(kx, kw, 1e-6, pos, d, 2), t)

    def prompt():
        ck, cv = fresh(n), fresh(n)
        sp, sm = torch.zeros((S, HK, n), dtype=torch.int32, device="cuda"), torch.zeros((S, HK, n), device="cuda")
        q = ops.qk_norm_rope(qg[:, :n], kg[:, :n], vg[:, :n], qwg, kwg, 1e-6, pg[:, :n], ck, cv, t, slot_pos=sp, slot_mass=sm, **opt)
        assert torch.equal(ck, all_k[:, :, :n]) and torch.equal(cv, all_v[:, :, :n]) and torch.equal(sp, pg[:, None, :n].expand(S, HK, n))
        assert torch.equal(q, q_rot[:, :, :n])
        mask = causal(1, W, n)
        weight = ops.attn_mass(q[:, :, n - W:], ck, mask.cuda(), t, scale)
        _, _, wm, em = attn_oracle(q[:, :, n - W:].cpu(), values(ck.cpu(), t), None, mask, scale, None, 0.0)
        assert ((weight.cpu().double() - wm).abs() <= em).all()
        past = torch.full((S,), n, dtype=torch.int32, device="cuda")
        bk, bv = fresh(budget), fresh(budget)
        kept, _, mo, po = ops.kv_evict(weight, sp, past, budget - 1, 4, 8, k=ck, v=cv, type_kv=t, k_out=bk[:, :, : budget - 1], v_out=bv[:, :, : budget - 1])
        want, _ = evict_oracle(weight.cpu().numpy(), sp.cpu().numpy(), [n] * S, [n] * S, budget - 1, 1, 4, 8)
        assert np.array_equal(kept.cpu().numpy(), want)
        mass, where = torch.zeros((S, HK, budget), device="cuda"), torch.zeros((S, HK, budget), dtype=torch.int32, device="cuda")
        mass[..., : budget - 1], where[..., : budget - 1] = mo, po
        return dict(k=bk, v=bv, mass=mass, pos=where, free=torch.full((S, HK, 1), budget - 1, dtype=torch.int32, device="cuda"),
                    q=qg[:, :1].clone(), kk=kg[:, :1].clone(), vv=vg[:, :1].clone(), at=pg[:, :1].clone(), past=torch.zeros(S, dtype=torch.int32, device="cuda"))

    def step(c):
        q = ops.qk_norm_rope(c["q"], c["kk"], c["vv"], qwg, kwg, 1e-6, c["at"], c["k"], c["v"], t, rows=c["free"], slot_pos=c["pos"], slot_mass=c["mass"], **opt)
        dst, _ = ops.flash_attn_ext_mass(q, c["k"], c["v"], None, t, scale, mass=c["mass"], decay=0.95, mass_out=c["mass"])
        _, out = ops.kv_evict(c["mass"], c["pos"], c["past"], budget - 1, 4, 8)
        c["free"].copy_(out)
        return q, dst

    def feed(c, i):
        for name, x in (("q", qg), ("kk", kg), ("vv", vg), ("at", pg)):
            c[name].copy_(x[:, n + i: n + i + 1])
        c["past"].fill_(n + i + 1)

    eager, replayed = prompt(), prompt()
    results = []
    for i in range(steps):
        feed(eager, i)
        old, free = eager["mass"].cpu(), eager["free"].cpu().long()
        q, dst = step(eager)
        old.scatter_(2, free, 0.0)
        k, v, p = (eager[x].cpu() for x in ("k", "v", "pos"))
        at = (torch.arange(S)[:, None, None], torch.arange(HK)[None, :, None], p.long())
        assert torch.equal(k, all_k.cpu()[at]) and torch.equal(v, all_v.cpu()[at])            # every slot holds the token that slot_pos names
        assert (torch.gather(p, 2, free) == n + i).all() and len({tuple(x) for x in p.reshape(-1, budget).tolist()}) >= 1
        assert all(len(set(x)) == budget for x in p.reshape(-1, budget).tolist())             # each token once
        wd, ed, wm, em = attn_oracle(q.cpu(), values(k, t), values(v, t), None, scale, old, 0.95)
        assert ((dst.cpu().double() - wd).abs() <= ed).all() and ((eager["mass"].cpu().double() - wm).abs() <= em).all()
        _, want = evict_oracle(eager["mass"].cpu().numpy(), p.numpy(), [n + i + 1] * S, [budget] * S, budget - 1, 1, 4, 8)
        assert np.array_equal(eager["free"].cpu().numpy(), want)
        assert not (torch.gather(p, 2, eager["free"].cpu().long()) < 4).any()                 # the sink stays
        results.append(dst.clone())

    feed(replayed, 0)
    saved = {x: y.clone() for x, y in replayed.items()}
    step(replayed)                                  # (a run before the capture, taken back)
    for x, y in saved.items():
        replayed[x].copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, dst = step(replayed)
    for i in range(steps):
        feed(replayed, i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dst, results[i])
    assert all(torch.equal(replayed[x], eager[x]) for x in ("k", "v", "mass", "pos", "free"))
