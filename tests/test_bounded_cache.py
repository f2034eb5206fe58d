"""Refusals of the bounded KV cache's entry points: every argument check answers before anything is launched, so no GPU is needed.
Pointers here are only ever compared with NULL and tested for alignment."""
import pytest

import llm_amd.blocks as B
import llm_amd.kernels as K

E_TYPE, E_SHAPE, E_ALIGN, E_NULL, E_WORKSPACE, E_UNSUPPORTED = -1, -2, -3, -4, -5, -6
P = 1 << 20        # a well-aligned address that is never followed


def store_args(**kw):
    a = K.QkNormRopeArgs()
    for f in ("q", "k", "v", "q_norm", "k_norm", "q_out", "k_out", "v_out", "rows", "pos", "slot_pos", "slot_mass"):
        setattr(a, f, P)
    for f in ("q", "k", "v", "qo", "ko", "vo"):
        for i, nb in enumerate((4096, 512, 1 << 16)):
            setattr(a, f"{f}_nb{i + 1}", nb)
    a.head_dim, a.dv, a.n_head, a.n_head_kv, a.n, a.ne3, a.n_rows = 128, 0, 8, 2, 1, 1, 16
    a.type_kv, a.n_dims, a.mode, a.n_ctx_orig = B.F16, 128, 2, 4096
    a.eps, a.freq_base, a.freq_scale, a.attn_factor, a.beta_fast, a.beta_slow = 1e-6, 1e4, 1.0, 1.0, 32.0, 1.0
    for f, v in kw.items():
        setattr(a, f, v)
    return a


@pytest.mark.parametrize("code, kw", [
    (E_NULL, dict(q=None)), (E_NULL, dict(k=None)), (E_NULL, dict(q_out=None)), (E_NULL, dict(k_out=None)), (E_NULL, dict(pos=None)),
    (E_NULL, dict(v=None)), (E_NULL, dict(v_out=None)),
    (E_UNSUPPORTED, dict(head_dim=0)), (E_UNSUPPORTED, dict(head_dim=100)), (E_UNSUPPORTED, dict(head_dim=264)), (E_UNSUPPORTED, dict(dv=12)),
    (E_UNSUPPORTED, dict(dv=512)), (E_UNSUPPORTED, dict(mode=8)), (E_UNSUPPORTED, dict(n_dims=20)),
    (E_SHAPE, dict(n_dims=136)), (E_SHAPE, dict(n_dims=-8)), (E_SHAPE, dict(n=-1)), (E_SHAPE, dict(ne3=-1)), (E_SHAPE, dict(n_head=0)),
    (E_SHAPE, dict(n_head_kv=0)), (E_SHAPE, dict(n_rows=-1)), (E_SHAPE, dict(n=1 << 25)), (E_SHAPE, dict(n=1 << 20, ne3=1 << 20)),
    (E_SHAPE, dict(freq_base=0.0)), (E_SHAPE, dict(freq_base=float("nan"))), (E_SHAPE, dict(freq_scale=0.0)), (E_SHAPE, dict(ext_factor=1.0, n_ctx_orig=0)),
    (E_SHAPE, dict(type_kv=B.Q8_0, head_dim=80, n_dims=80)), (E_SHAPE, dict(type_kv=B.Q4_0, dv=72)),
    (E_TYPE, dict(type_kv=B.Q4_K)), (E_TYPE, dict(type_kv=B.I32)),
    (E_ALIGN, dict(q=P + 4)), (E_ALIGN, dict(k_nb2=520)), (E_ALIGN, dict(q_out=P + 8)), (E_ALIGN, dict(q_norm=P + 4)), (E_ALIGN, dict(k_out=P + 2)),
    (E_ALIGN, dict(vo_nb1=264)), (E_ALIGN, dict(type_kv=B.Q8_0, k_out=P + 1)), (E_ALIGN, dict(pos=P + 2)), (E_ALIGN, dict(rows_nb2=6)),
    (E_ALIGN, dict(slot_mass=P + 1)),
])
def test_qk_norm_rope_refuses(code, kw):
    assert K.lib.mi355_qk_norm_rope(store_args(**kw), None) == code


@pytest.mark.parametrize("kw", [
    dict(q_out=P + 512), dict(q_out=P - 512), dict(q_out=P, qo_nb2=1024), dict(q_out=P, n=4, qo_nb1=512, qo_nb2=2048), dict(q_out=P, ne3=2, qo_nb3=1 << 15),
    dict(q_out=9 * P), dict(q_out=10 * P + 512), dict(q_out=9 * P - 3584), dict(q_out=P + 32, n=3), dict(q_out=P, n_head=2, ne3=2, q_nb3=1024, qo_nb2=1024, qo_nb3=512),
])
def test_qk_norm_rope_refuses_q_out_over_its_inputs(kw):
    """in place means row for row; any other order would overwrite rows that are still to be read"""
    assert K.lib.mi355_qk_norm_rope(store_args(**{**dict(k=9 * P, v=10 * P), **kw}), None) == E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(qo_nb2=0), dict(qo_nb2=256), dict(n=2, qo_nb1=0), dict(n=2, qo_nb1=2048), dict(ne3=2, qo_nb3=0), dict(ko_nb2=0), dict(ko_nb1=128), dict(ko_nb1=0),
                                dict(ne3=2, ko_nb3=0), dict(vo_nb2=240), dict(ne3=2, vo_nb3=4096), dict(type_kv=B.Q8_0, vo_nb1=134, vo_nb2=4096)])
def test_qk_norm_rope_refuses_outputs_that_share_memory_with_themselves(kw):
    """an expanded tensor: several rows in one place"""
    assert K.lib.mi355_qk_norm_rope(store_args(**{**dict(q_out=9 * P, k_out=10 * P, v_out=12 * P, rows=None, n=2), **kw}), None) == E_UNSUPPORTED


def test_qk_norm_rope_of_nothing_launches_nothing():
    assert K.lib.mi355_qk_norm_rope(None, None) == E_NULL
    assert K.lib.mi355_qk_norm_rope(store_args(n=0), None) == 0
    assert K.lib.mi355_qk_norm_rope(store_args(ne3=0), None) == 0


def test_qk_norm_rope_of_tensors_without_an_address():
    none = dict(q=None, k=None, v=None, q_out=None, k_out=None, v_out=None, pos=None, rows=None)
    assert K.lib.mi355_qk_norm_rope(store_args(ne3=0, **none), None) == 0 and K.lib.mi355_qk_norm_rope(store_args(n=0, **none), None) == 0
    assert K.lib.mi355_qk_norm_rope(store_args(n_rows=0, q=None), None) == E_NULL


def evict_args(**kw):
    a = K.KvEvictArgs()
    for i, f in enumerate(("mass", "slot_pos", "n_past", "kept", "evicted", "k", "v", "k_out", "v_out", "mass_out", "pos_out")):
        setattr(a, f, P * (i + 1))
    for f in ("mass", "pos", "kept", "ev", "k", "v", "ko", "vo", "mo", "po"):
        setattr(a, f + "_nb2", 4096)
        setattr(a, f + "_nb3", 1 << 16)
        if f in ("k", "v", "ko", "vo"):
            setattr(a, f + "_nb1", 256)
    a.n_kv, a.n_keep, a.n_evict, a.n_head_kv, a.ne3, a.d, a.dv, a.type_kv = 100, 50, 50, 2, 1, 128, 0, B.F16
    for f, v in kw.items():
        setattr(a, f, v)
    return a


@pytest.mark.parametrize("code, kw", [
    (E_NULL, dict(mass=None)), (E_NULL, dict(slot_pos=None)), (E_NULL, dict(n_past=None)), (E_NULL, dict(kept=None)), (E_NULL, dict(k=None)),
    (E_NULL, dict(v_out=None)),
    (E_SHAPE, dict(n_kv=-1)), (E_SHAPE, dict(n_kv=1 << 32)), (E_SHAPE, dict(n_kv=(1 << 30) + 1)), (E_SHAPE, dict(n_keep=(1 << 30) + 1)), (E_SHAPE, dict(n_evict=(1 << 30) + 1)), (E_SHAPE, dict(n_keep=0)), (E_SHAPE, dict(n_evict=-1)), (E_SHAPE, dict(n_sink=-1)),
    (E_SHAPE, dict(n_sink=26, n_recent=25)), (E_SHAPE, dict(n_recent=51)), (E_SHAPE, dict(n_sink=2 ** 31 - 1, n_recent=2 ** 31 - 1)),
    (E_SHAPE, dict(n_head_kv=0)), (E_SHAPE, dict(ne3=-1)), (E_SHAPE, dict(ne3=65536)), (E_SHAPE, dict(d=0)), (E_SHAPE, dict(type_kv=B.Q8_0, d=40)),
    (E_SHAPE, dict(type_kv=B.Q4_0, dv=8)), (E_TYPE, dict(type_kv=B.Q4_K)), (E_TYPE, dict(type_kv=99)),
    (E_ALIGN, dict(mass=P + 2)), (E_ALIGN, dict(kept_nb2=6)), (E_ALIGN, dict(k_out=P + 1)), (E_ALIGN, dict(v_nb1=257)),
    (E_UNSUPPORTED, dict(k_out=6 * P)), (E_UNSUPPORTED, dict(v_out=7 * P)), (E_UNSUPPORTED, dict(mass_out=P)), (E_UNSUPPORTED, dict(pos_out=2 * P)),
])
def test_kv_evict_refuses(code, kw):
    assert K.lib.mi355_kv_evict(evict_args(**kw), None) == code


# caches of 100 slots x 256 bytes: slot-major (pitch 512: K and V of a slot side by side, heads 100 slots apart) and head-major ones
SIDE = dict(k_nb1=512, v_nb1=512, v=6 * P + 256, k_nb2=51200, v_nb2=51200, ko_nb2=51200, vo_nb2=51200)


@pytest.mark.parametrize("kw", [
    dict(k_out=6 * P + 256), dict(k_out=6 * P + 25600 - 256, k_nb2=25600), dict(k_out=6 * P - 49 * 256), dict(k_out=7 * P + 2, v_nb1=258), dict(v_out=6 * P + 4096),
    dict(k_out=6 * P + (1 << 16), ne3=2), dict(k_out=8 * P, v_out=8 * P + 128), dict(k_out=8 * P, v_out=8 * P), dict(mass_out=P + 196), dict(mass_out=P - 100),
    dict(pos_out=2 * P + 4096 + 200), dict(pos_out=P + 4), dict(kept=P + 8), dict(evicted=2 * P + 4), dict(kept=3 * P), dict(n_used=5 * P, evicted=5 * P),
    dict(mass_out=10 * P, pos_out=10 * P + 100), dict(evicted=4 * P + 100), dict(kept=6 * P + 4), dict(mass_out=9 * P + 1000),
    dict(SIDE, k_out=6 * P + 256, ko_nb1=512), dict(SIDE, k_out=6 * P + 128, ko_nb1=512), dict(SIDE, k_out=6 * P, ko_nb1=512), dict(SIDE, k_out=6 * P + 4, ko_nb1=516),
    dict(k_nb1=-256, k_out=6 * P - 99 * 256), dict(k_nb2=-25600, k_out=6 * P - 25600),
])
def test_kv_evict_refuses_outputs_that_meet_what_it_reads(kw):
    """a gathered row read after its place has been written: any byte in common, wherever the views begin"""
    assert K.lib.mi355_kv_evict(evict_args(**kw), None) == E_UNSUPPORTED


NEST = dict(k_nb1=256, k_nb2=25600, k_nb3=51200, v_nb2=25600, v_nb3=51200, ko_nb2=12800, ko_nb3=25600, vo_nb2=12800, vo_nb3=25600)


@pytest.mark.parametrize("kw", [dict(ko_nb2=0), dict(ko_nb1=0), dict(ko_nb1=128), dict(ko_nb2=12544), dict(ne3=2, ko_nb3=0), dict(vo_nb1=254), dict(ne3=2, vo_nb3=12800), dict(kept_nb2=0),
                                dict(kept_nb2=196), dict(ev_nb2=100), dict(mo_nb2=0), dict(po_nb2=4), dict(ne3=2, mo_nb3=4000)])
def test_kv_evict_refuses_outputs_that_share_memory_with_themselves(kw):
    assert K.lib.mi355_kv_evict(evict_args(**{**NEST, **kw}), None) == E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(n_keep=1 << 30), dict(n_keep=1 << 28), dict(n_keep=1 << 29, k_nb1=258), dict(n_keep=1 << 28, ne3=0)])
def test_kv_evict_refuses_more_rows_than_a_grid_holds(kw):
    """before the first of its launches, not by the second's failure"""
    far = {f: 1 << (50 + i) for i, f in enumerate(("k", "v", "k_out", "v_out", "mass_out", "pos_out", "kept", "evicted"))}
    assert K.lib.mi355_kv_evict(evict_args(**far, **kw), None) == E_SHAPE


def test_kv_evict_of_no_sequences_launches_nothing():
    assert K.lib.mi355_kv_evict(None, None) == E_NULL
    assert K.lib.mi355_kv_evict(evict_args(ne3=0), None) == 0


def test_kv_evict_of_tensors_without_an_address():
    assert K.lib.mi355_kv_evict(evict_args(ne3=0, mass=None, slot_pos=None, n_past=None, kept=None, evicted=None, k=None, v=None, k_out=None, v_out=None,
                                           mass_out=None, pos_out=None), None) == 0
    assert K.lib.mi355_kv_evict(evict_args(ne3=0, n_keep=0), None) == E_SHAPE


def attn_args(**kw):
    a, w = K.FattnArgs(), K.AttnMassArgs()
    for f in ("q", "k", "v", "mask", "dst"):
        setattr(a, f, P)
    for f in ("q", "k", "v", "m", "d"):
        for i, nb in enumerate((512, 4096, 1 << 16)):
            setattr(a, f"{f}_nb{i + 1}", nb)
    a.type_k = a.type_v = B.F16
    a.d, a.n_q, a.n_kv, a.n_head, a.n_head_kv, a.ne3, a.dv, a.m_ne2, a.m_ne3, a.scale = 128, 1, 64, 8, 2, 1, 0, 1, 1, 0.1
    w.mass_in = w.mass_out = P
    w.in_nb2 = w.out_nb2 = 256
    w.in_nb3 = w.out_nb3 = 1024
    w.decay = 1.0
    for f, v in kw.items():
        setattr(w if f in ("mass_in", "mass_out", "in_nb2", "out_nb3", "decay") else a, f, v)
    return a, w


BOTH = [
    (E_NULL, dict(q=None)), (E_NULL, dict(k=None)), (E_NULL, dict(mass_out=None)),
    (E_UNSUPPORTED, dict(d=0)), (E_UNSUPPORTED, dict(d=100)), (E_UNSUPPORTED, dict(d=512)),
    (E_TYPE, dict(type_k=B.F32, type_v=B.F32)), (E_TYPE, dict(type_k=B.Q4_K, type_v=B.Q4_K)),
    (E_SHAPE, dict(type_k=B.Q8_0, type_v=B.Q8_0, d=80)), (E_SHAPE, dict(n_head=0)), (E_SHAPE, dict(n_head_kv=3)), (E_SHAPE, dict(n_head_kv=0)),
    (E_SHAPE, dict(n_q=0)), (E_SHAPE, dict(n_q=65536)), (E_SHAPE, dict(n_kv=-1)), (E_SHAPE, dict(n_kv=1 << 31)), (E_SHAPE, dict(ne3=0)),
    (E_SHAPE, dict(m_ne2=0)), (E_SHAPE, dict(m_ne3=0)), (E_SHAPE, dict(n_head=65536, n_head_kv=1)), (E_SHAPE, dict(n_head=65535, n_head_kv=1, n_q=2)),
    (E_SHAPE, dict(k_nb1=-512)), (E_SHAPE, dict(k_nb1=1 << 31)), (E_SHAPE, dict(m_ne2=65536)), (E_SHAPE, dict(m_ne2=1000, m_ne3=1000)), (E_SHAPE, dict(m_ne3=1 << 62, m_ne2=4)),
    (E_ALIGN, dict(q=P + 4)), (E_ALIGN, dict(q_nb1=520)), (E_ALIGN, dict(k=P + 8)), (E_ALIGN, dict(k_nb1=264)), (E_ALIGN, dict(mask=P + 1)),
    (E_ALIGN, dict(m_nb1=511)), (E_ALIGN, dict(mass_in=P + 2)), (E_ALIGN, dict(out_nb3=1022)), (E_ALIGN, dict(type_k=B.Q4_0, type_v=B.Q4_0, k_nb2=4097)),
]


@pytest.mark.parametrize("code, kw", BOTH + [
    (E_NULL, dict(v=None)), (E_NULL, dict(dst=None)), (E_UNSUPPORTED, dict(dv=136)), (E_UNSUPPORTED, dict(dv=12)), (E_TYPE, dict(type_v=B.BF16)),
    (E_SHAPE, dict(type_k=B.Q8_0, type_v=B.Q8_0, dv=40)), (E_UNSUPPORTED, dict(n_q=9)), (E_ALIGN, dict(v_nb3=8)), (E_ALIGN, dict(dst=P + 4)),
    (E_SHAPE, dict(v_nb1=1 << 31)), (E_SHAPE, dict(v_nb1=-512)),
])
def test_flash_attn_ext_mass_refuses(code, kw):
    assert K.lib.mi355_flash_attn_ext_mass(*attn_args(**kw), P, 1 << 40, None) == code


@pytest.mark.parametrize("code, kw", BOTH)
def test_attn_mass_refuses(code, kw):
    assert K.lib.mi355_attn_mass(*attn_args(**{k: v for k, v in kw.items()}), P, 1 << 40, None) == code


@pytest.mark.parametrize("kw", [dict(mass_in=P + 4), dict(mass_in=P - 252), dict(mass_in=P, in_nb2=512), dict(mass_in=P + 256), dict(mass_in=P + 1024, ne3=2)])
@pytest.mark.parametrize("fn", [K.lib.mi355_flash_attn_ext_mass, K.lib.mi355_attn_mass])
def test_attention_mass_refuses_a_shifted_table(fn, kw):
    assert fn(*attn_args(**kw), P, 1 << 40, None) == E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(out_nb2=0), dict(out_nb2=252), dict(ne3=2, out_nb3=0), dict(ne3=2, out_nb3=256)])
@pytest.mark.parametrize("fn", [K.lib.mi355_flash_attn_ext_mass, K.lib.mi355_attn_mass])
def test_attention_mass_refuses_an_expanded_table(fn, kw):
    a, w = attn_args(**{k: v for k, v in kw.items() if k != "out_nb2"}, mass_in=None)
    w.out_nb2 = kw.get("out_nb2", 256)
    assert fn(a, w, 9 * P, 1 << 40, None) == E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(d_nb1=0), dict(d_nb1=256), dict(n_q=2, d_nb2=0), dict(ne3=2, d_nb3=0)])
def test_flash_attn_ext_mass_refuses_an_expanded_dst(kw):
    a, w = attn_args(**kw, mass_in=None)
    assert K.lib.mi355_flash_attn_ext_mass(a, w, 9 * P, 1 << 40, None) == E_UNSUPPORTED


def test_attention_mass_workspaces():
    for fn, size in ((K.lib.mi355_flash_attn_ext_mass, K.lib.mi355_flash_attn_ext_mass_workspace_bytes), (K.lib.mi355_attn_mass, K.lib.mi355_attn_mass_workspace_bytes)):
        assert fn(None, None, P, 1 << 40, None) == E_NULL and size(None) == -1
        for kw in (dict(), dict(n_q=7, n_kv=5000, ne3=3), dict(n_kv=100000, n_head=64, n_head_kv=8)):
            a, w = attn_args(**kw)
            need = size(a)
            assert need >= 0
            if need > 0:
                assert fn(a, w, P, need - 1, None) == E_WORKSPACE and fn(a, w, None, 0, None) == E_WORKSPACE
                assert fn(a, w, P + 4, need, None) == E_ALIGN
    assert K.lib.mi355_attn_mass_workspace_bytes(attn_args(n_q=-1)[0]) == -1
    assert K.lib.mi355_attn_mass_workspace_bytes(attn_args(n_q=100, m_ne2=0)[0]) == -1
    assert K.lib.mi355_attn_mass_workspace_bytes(attn_args(n_q=100, m_ne2=0, mask=None)[0]) > 0


@pytest.mark.parametrize("n_kv", [0, 200, 512, 100000])
@pytest.mark.parametrize("kw", [dict(n_q=0), dict(n_q=0, d=256), dict(ne3=0), dict(n_q=0, mask=None)])
def test_attention_mass_workspaces_of_no_queries(n_kv, kw):
    """answered, not divided by: the size is asked for before the call itself can refuse"""
    a, w = attn_args(n_kv=n_kv, **kw)
    for size, run in ((K.lib.mi355_flash_attn_ext_mass_workspace_bytes, K.lib.mi355_flash_attn_ext_mass), (K.lib.mi355_attn_mass_workspace_bytes, K.lib.mi355_attn_mass)):
        assert size(a) == -1 and run(a, w, P, 1 << 40, None) == E_SHAPE


@pytest.mark.parametrize("kw", [dict(n_q=65535, n_head=64, n_head_kv=8, ne3=65), dict(n_q=65535, n_kv=1 << 20, m_ne2=2), dict(n_q=60000, n_head=16, n_kv=1 << 20, m_ne3=10, ne3=10)])
def test_attn_mass_refuses_more_than_a_grid_holds(kw):
    a, w = attn_args(**kw)
    assert K.lib.mi355_attn_mass_workspace_bytes(a) == -1 and K.lib.mi355_attn_mass(a, w, P, 1 << 62, None) == E_SHAPE


@pytest.mark.parametrize("kw", [dict(n_head=65535, n_head_kv=65535, n_q=8, ne3=65535, n_kv=1 << 30), dict(n_head=60000, n_head_kv=60000, ne3=60000, n_kv=1 << 30),
                                dict(n_q=1 << 40), dict(n_kv=1 << 40), dict(ne3=1 << 40), dict(n_q=100, m_ne2=1 << 20, m_ne3=1 << 20)])
def test_attention_mass_workspaces_past_64_bits(kw):
    """a size whose product would wrap is refused by the size and by the call"""
    a, w = attn_args(**kw)
    for size, run in ((K.lib.mi355_flash_attn_ext_mass_workspace_bytes, K.lib.mi355_flash_attn_ext_mass), (K.lib.mi355_attn_mass_workspace_bytes, K.lib.mi355_attn_mass)):
        assert size(a) == -1 and run(a, w, P, 1 << 62, None) in (E_SHAPE, E_UNSUPPORTED)


def test_library_and_torch_share_one_hip_runtime():
    """whichever is imported first: two runtimes in a process refuse each other's device"""
    import os
    import subprocess
    import sys
    code = ("import llm_amd.kernels, torch\n"
            "libs = {l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l}\n"
            "assert len(libs) == 1, libs")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
