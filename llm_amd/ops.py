"""Host-side mirror of the reference's operator interface for the hot path, on torch device tensors.

Same names and argument meaning as the ggml ops the backend serves (ggml/include/ggml.h):
  mul_mat(a, b)            ggml_mul_mat      a = weights [M rows of K] (block-quantized bytes), b = [N, K] f32 -> [N, M] f32
  mul_mat_id(as_, b, ids)  ggml_mul_mat_id
plus the two contract-level primitives quantize_q8_1 / dequantize.  Everything runs through the C ABI
of libmi355_kernels.so on the current torch stream; torch only owns the memory.
"""
import torch

from . import blocks as B
from . import kernels as K


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _u8(t):
    assert t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous()
    return t


def _dst_rows(dst):
    return dst.stride(0) if dst.dim() > 1 else dst.numel()


def quantize_q8_1(x):
    """x: [..., K] f32 (last dim contiguous, up to 4-D) -> uint8 [rows, K/32*36] of block_q8_1."""
    assert x.is_cuda and x.dtype == torch.float32 and x.stride(-1) == 1 and 1 <= x.dim() <= 4
    k = x.shape[-1]
    shp = [1] * (4 - x.dim()) + list(x.shape)
    st = [0] * (4 - x.dim()) + list(x.stride())
    ne3, ne2, ne1 = shp[0], shp[1], shp[2]
    nb3, nb2, nb1 = (s * 4 for s in st[:3])
    rows = ne1 * ne2 * ne3
    y = torch.empty((rows, k // 32 * 36), dtype=torch.uint8, device=x.device)
    K.check(K.lib.mi355_quantize_row_q8_1(x.data_ptr(), y.data_ptr(), k, ne1, ne2, ne3, nb1, nb2, nb3, _stream()),
            "mi355_quantize_row_q8_1")
    return y


def quantize_act(x):
    """x: [rows, K] f32 contiguous -> (act_q int8 [rows, K], act_ds f32 [rows, K/32, 2])."""
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.is_contiguous()
    rows, k = x.shape
    aq = torch.empty((rows, k), dtype=torch.int8, device=x.device)
    ads = torch.empty((rows, k // 32, 2), dtype=torch.float32, device=x.device)
    K.check(K.lib.mi355_quantize_act(x.data_ptr(), aq.data_ptr(), ads.data_ptr(), k, rows, 1, 1, k * 4, 0, 0, _stream()),
            "mi355_quantize_act")
    return aq, ads


def dequantize(t, blocks, n):
    """blocks: uint8 device tensor holding n elements of type t -> f32 [n]."""
    _u8(blocks)
    assert blocks.numel() >= B.row_size(t, n)
    y = torch.empty(n, dtype=torch.float32, device=blocks.device)
    K.check(K.lib.mi355_dequantize_row(t, blocks.data_ptr(), y.data_ptr(), n, _stream()), "mi355_dequantize_row")
    return y


def mul_mat_vec_q(t, w, m, k, aq, ads, ncols, dst=None, w_row_stride=None, residual=None, sum_out=None):
    """Decode mat-vec on pre-quantized activations (act rows 0..ncols-1).  residual ([ncols, m] f32): also store
    sum_out = result + residual (sum_out may be dst -> only the sum is stored, or residual itself)."""
    _u8(w)
    if dst is None:
        dst = torch.empty((ncols, m), dtype=torch.float32, device=w.device)
    a = K.MmvqArgs()
    a.type, a.W, a.w_row_stride, a.w_ch_stride = t, w.data_ptr(), w_row_stride or B.row_size(t, k), 0
    a.act_q, a.act_ds, a.act_ch_stride = aq.data_ptr(), ads.data_ptr(), 0
    a.dst, a.dst_col_stride, a.dst_ch_stride = dst.data_ptr(), dst.stride(0), 0
    a.m, a.k, a.ncols, a.nchannels, a.ch_ratio = m, k, ncols, 1, 1
    if residual is not None:
        a.residual, a.sum = residual.data_ptr(), sum_out.data_ptr()
    K.check(K.lib.mi355_mul_mat_vec_q(a, _stream()), "mi355_mul_mat_vec_q")
    return dst


def mul_mat_vec_q_group(t, ws, ms, k, aq, ads, ncols):
    """Grouped decode mat-vec: several weight matrices (same type and k) on the same pre-quantized activations in
    ONE launch (mi355_mul_mat_vec_q_group).  ws: list of uint8 block tensors, ms: rows of each -> list of [ncols, m]."""
    outs, arr = [], (K.MmvqArgs * len(ws))()
    for i, (w, m) in enumerate(zip(ws, ms)):
        _u8(w)
        dst = torch.empty((ncols, m), dtype=torch.float32, device=w.device)
        a = arr[i]
        a.type, a.W, a.w_row_stride, a.w_ch_stride = t, w.data_ptr(), B.row_size(t, k), 0
        a.act_q, a.act_ds, a.act_ch_stride = aq.data_ptr(), ads.data_ptr(), 0
        a.dst, a.dst_col_stride, a.dst_ch_stride = dst.data_ptr(), dst.stride(0), 0
        a.m, a.k, a.ncols, a.nchannels, a.ch_ratio = m, k, ncols, 1, 1
        outs.append(dst)
    K.check(K.lib.mi355_mul_mat_vec_q_group(arr, len(ws), _stream()), "mi355_mul_mat_vec_q_group")
    return outs


def act_bf16(b):
    """f32 [n, k] (row stride free, 16-byte aligned) -> bf16 [n, k] as uint16 (mi355_act_bf16)."""
    assert b.is_cuda and b.dtype == torch.float32 and b.dim() == 2 and b.stride(1) == 1
    n, k = b.shape
    y = torch.empty((n, k), dtype=torch.int16, device=b.device)
    K.check(K.lib.mi355_act_bf16(b.data_ptr(), y.data_ptr(), k, n, 1, 1, b.stride(0) * 4, 0, 0, _stream()), "mi355_act_bf16")
    return y


def mul_mat_dq(t, w, b, m):
    """Prefill GEMM through the dequantize-in-LDS bf16 MFMA kernel: b = [n, k] f32 -> [n, m] f32."""
    _u8(w)
    n, k = b.shape
    y = act_bf16(b)
    dst = torch.empty((n, m), dtype=torch.float32, device=b.device)
    K.check(K.mul_mat_dq(t, w.data_ptr(), B.row_size(t, k), y.data_ptr(), k, dst.data_ptr(), m, m, k, n,
                                   _stream()), "mi355_mul_mat_dq")
    return dst


def mul_mat(t, w, b, m, workspace=None):
    """ggml_mul_mat: w = [m rows] blocks of type t (uint8), b = [n, k] f32 -> [n, m] f32."""
    _u8(w)
    assert b.is_cuda and b.dtype == torch.float32 and b.dim() == 2 and b.is_contiguous()
    n, k = b.shape
    need = K.lib.mi355_mul_mat_workspace_bytes(k, n)
    if workspace is None:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=b.device)
    dst = torch.empty((n, m), dtype=torch.float32, device=b.device)
    K.check(K.lib.mi355_mul_mat(t, w.data_ptr(), B.row_size(t, k), b.data_ptr(), dst.data_ptr(), m, k, n,
                                workspace.data_ptr(), workspace.numel(), _stream()), "mi355_mul_mat")
    return dst


def mul_mat_id(t, as_, b, ids, m, n_expert):
    """ggml_mul_mat_id for decode-sized batches: as_ = [n_expert][m rows] blocks, b = [n_tokens, b_ne1, k] f32,
    ids = [n_tokens, n_used] int32 (device) -> [n_tokens, n_used, m] f32."""
    _u8(as_)
    assert b.dim() == 3 and b.is_contiguous() and ids.dtype == torch.int32 and ids.dim() == 2
    n_tok, b_ne1, k = b.shape
    n_used = ids.shape[1]
    aq, ads = quantize_act(b.reshape(n_tok * b_ne1, k))
    dst = torch.empty((n_tok, n_used, m), dtype=torch.float32, device=b.device)
    a = K.MmvqArgs()
    rs = B.row_size(t, k)
    a.type, a.W, a.w_row_stride, a.w_ch_stride = t, as_.data_ptr(), rs, rs * m
    a.act_q, a.act_ds, a.act_ch_stride = aq.data_ptr(), ads.data_ptr(), b_ne1
    a.dst, a.dst_col_stride, a.dst_ch_stride = dst.data_ptr(), m, m
    a.m, a.k, a.ncols, a.nchannels, a.ch_ratio = m, k, 1, n_tok * n_used, 1
    a.ids, a.ids_stride, a.ids_nused, a.act_ne1, a.n_expert = ids.data_ptr(), ids.stride(0), n_used, b_ne1, n_expert
    K.check(K.lib.mi355_mul_mat_vec_q(a, _stream()), "mi355_mul_mat_vec_q(ids)")
    return dst


def flash_attn_ext(q, k, v, mask, type_kv, n_kv, scale, max_bias=0.0, logit_softcap=0.0, use_workspace=True, quant=False,
                   workspace_bytes=None, noalloc=False, bf16=False, dv=None):
    """ggml_flash_attn_ext, batch 1.  q: [n_head, n_q, d] f32; k, v: [n_head_kv, n_kv, row_bytes] uint8 rows of
    type_kv (F16 / BF16 / Q8_0 / Q4_0); mask: [n_q_pad, n_kv] f16 bits (int16) or None -> [n_q, n_head, dv] f32 (dv: V's head size
    where it differs from d, e.g. 192 / 128)."""
    assert q.is_cuda and q.dtype == torch.float32 and q.is_contiguous() and k.is_contiguous() and v.is_contiguous()
    n_head, n_q, d = q.shape
    n_head_kv = k.shape[0]
    d_k, d = d, (dv if dv else d)          # below, d is the head size of V and dst
    dst = torch.empty((n_q, n_head, d), dtype=torch.float32, device=q.device)
    a = K.FattnArgs()
    a.q, a.q_nb1, a.q_nb2, a.q_nb3 = q.data_ptr(), d_k * 4, n_q * d_k * 4, n_head * n_q * d_k * 4
    rb = k.shape[2] * k.element_size()
    a.k, a.type_k, a.k_nb1, a.k_nb2, a.k_nb3 = k.data_ptr(), type_kv, rb, rb * k.shape[1], rb * k.shape[1] * n_head_kv
    rb = v.shape[2] * v.element_size()
    a.v, a.type_v, a.v_nb1, a.v_nb2, a.v_nb3 = v.data_ptr(), type_kv, rb, rb * v.shape[1], rb * v.shape[1] * n_head_kv
    if mask is not None:
        assert mask.is_contiguous() and mask.element_size() == 2
        a.mask, a.m_nb1, a.m_nb2, a.m_nb3, a.m_ne2, a.m_ne3 = mask.data_ptr(), mask.shape[1] * 2, mask.numel() * 2, mask.numel() * 2, 1, 1
    a.dst, a.d_nb1, a.d_nb2, a.d_nb3 = dst.data_ptr(), d * 4, n_head * d * 4, n_q * n_head * d * 4
    a.d, a.n_q, a.n_kv, a.n_head, a.n_head_kv, a.ne3 = d_k, n_q, n_kv, n_head, n_head_kv, 1
    a.dv = d if dv else 0
    a.scale, a.max_bias, a.logit_softcap = scale, max_bias, logit_softcap
    ws, wsb = None, 0
    if noalloc:      # the entry point that allocates nothing: the split-KV scratch is a fixed array inside the library
        K.check(K.lib.mi355_flash_attn_ext_noalloc(a, _stream()), "mi355_flash_attn_ext_noalloc")
        return dst
    if use_workspace:
        wsb = workspace_bytes if workspace_bytes is not None else K.lib.mi355_flash_attn_ext_workspace_bytes(a)
        ws = torch.zeros(max(wsb, 16), dtype=torch.uint8, device=q.device)   # arrival counters must start at zero
    if quant:
        aq = torch.empty((n_q, n_head * d), dtype=torch.int8, device=q.device)
        ads = torch.empty((n_q, n_head * d // 32, 2), dtype=torch.float32, device=q.device)
        for _ in range(2):   # twice on the same workspace: the counters must have returned to zero
            K.check(K.lib.mi355_flash_attn_ext_quant(a, ws.data_ptr() if ws is not None else None, wsb, aq.data_ptr(), ads.data_ptr(),
                                                     _stream()), "mi355_flash_attn_ext_quant")
        return dst, aq, ads
    if bf16:         # prefill: the bf16 rows of the result from the same launch
        abf = torch.empty((n_q, n_head * d), dtype=torch.int16, device=q.device)
        K.check(K.lib.mi355_flash_attn_ext_bf16(a, ws.data_ptr() if ws is not None else None, wsb, abf.data_ptr(), _stream()), "mi355_flash_attn_ext_bf16")
        return dst, abf
    K.check(K.lib.mi355_flash_attn_ext(a, ws.data_ptr() if ws is not None else None, wsb, _stream()), "mi355_flash_attn_ext")
    return dst


def rope(x, pos, n_dims, mode, n_ctx_orig=8192, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0,
         beta_fast=32.0, beta_slow=1.0, freq_factors=None):
    """ggml_rope_ext on x = [n_tokens, n_head, head_dim] f32 (contiguous), pos = [n_tokens] int32."""
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous() and pos.dtype == torch.int32
    dst = torch.empty_like(x)
    tx, td = K.Tensor.of(x), K.Tensor.of(dst)
    K.check(K.lib.mi355_rope_f32(tx, pos.data_ptr(), freq_factors.data_ptr() if freq_factors is not None else None, td, n_dims, mode,
                                 n_ctx_orig, freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow, _stream()), "mi355_rope_f32")
    return dst


def qkv_rope_matvec(type_qk, type_v, wq, wk, wv, m_q, m_k, m_v, k, aq, ads, pos, head_dim, n_dims, mode, kv_dtype=torch.float16,
                    n_ctx_orig=8192, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
                    beta_slow=1.0, freq_factors=None, type_k=None, norm=None):
    """Fused decode attention input (mi355_qkv_rope_matvec): -> (q f32 [m_q], k [m_k], v [m_v] of kv_dtype).
    type_k: type of wk when it differs from wq's (type_qk)."""
    q = torch.empty(m_q, dtype=torch.float32, device=wq.device)
    ko = torch.empty(m_k, dtype=kv_dtype, device=wq.device)
    vo = torch.empty(m_v, dtype=kv_dtype, device=wq.device)
    a = K.QkvRopeArgs()
    a.type_qk, a.type_v, a.wq, a.wk, a.wv = type_qk, type_v, wq.data_ptr(), wk.data_ptr(), wv.data_ptr()
    a.wq_row_stride = B.row_size(type_qk, k)
    a.wk_row_stride = B.row_size(type_k if type_k is not None else type_qk, k)
    a.type_k = type_k if type_k is not None and type_k != type_qk else 0
    a.wv_row_stride = B.row_size(type_v, k)
    a.m_q, a.m_k, a.m_v, a.k = m_q, m_k, m_v, k
    a.q_out, a.k_out, a.v_out = q.data_ptr(), ko.data_ptr(), vo.data_ptr()
    if norm is not None:     # (x [k], w [k], eps, out [k]): rms_norm(x) * w computed inside the launch, aq / ads unused
        a.norm_x, a.norm_w, a.norm_eps, a.norm_out = norm[0].data_ptr(), norm[1].data_ptr(), norm[2], norm[3].data_ptr()
    else:
        a.act_q, a.act_ds = aq.data_ptr(), ads.data_ptr()
    a.k_out_type = a.v_out_type = B.F16 if kv_dtype == torch.float16 else B.F32
    a.pos, a.freq_factors = pos.data_ptr(), freq_factors.data_ptr() if freq_factors is not None else None
    a.head_dim, a.n_dims, a.mode, a.n_ctx_orig = head_dim, n_dims, mode, n_ctx_orig
    a.freq_base, a.freq_scale, a.ext_factor, a.attn_factor, a.beta_fast, a.beta_slow = freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow
    K.check(K.lib.mi355_qkv_rope_matvec(a, _stream()), "mi355_qkv_rope_matvec")
    return q, ko, vo


def glu_matvec(t, w_gate, w_up, m, k, aq, ads, glu_op=2, quant=True, keep=True, norm=None, ids=None, n_expert=0):
    """Fused decode feed-forward input (mi355_glu_matvec): -> (dst f32 [m], gate f32 [m] | None, up f32 [m] | None,
    out_q int8 [m] | None, out_ds f32 [m/32, 2] | None).  norm = (x [k] f32, w [k] f32, eps, out [k] f32): the
    activations are rms_norm(x) * w, computed inside the launch (aq / ads unused, may be None)."""
    _u8(w_gate); _u8(w_up)
    dev = w_gate.device
    ns = 1 if ids is None else ids.numel()       # ids: int32 [n_slots] expert of each slot; w_gate / w_up then hold n_expert matrices
    dst = torch.full((ns * m,), float("nan"), dtype=torch.float32, device=dev)
    g = torch.full((ns * m,), float("nan"), dtype=torch.float32, device=dev) if keep else None
    u = torch.full((ns * m,), float("nan"), dtype=torch.float32, device=dev) if keep else None
    oq = torch.zeros(ns * m, dtype=torch.int8, device=dev) if quant else None
    ods = torch.zeros((ns * m // 32, 2), dtype=torch.float32, device=dev) if quant else None
    a = K.GluMatvecArgs()
    a.type, a.glu_op, a.w_gate, a.w_up = t, glu_op, w_gate.data_ptr(), w_up.data_ptr()
    a.gate_row_stride = a.up_row_stride = B.row_size(t, k)
    a.m, a.k = m, k
    if norm is not None:
        a.norm_x, a.norm_w, a.norm_eps, a.norm_out = norm[0].data_ptr(), norm[1].data_ptr(), norm[2], norm[3].data_ptr()
    else:
        a.act_q, a.act_ds = aq.data_ptr(), ads.data_ptr()
    a.gate_out, a.up_out, a.dst = g.data_ptr() if keep else None, u.data_ptr() if keep else None, dst.data_ptr()
    a.out_q, a.out_ds = oq.data_ptr() if quant else None, ods.data_ptr() if quant else None
    if ids is not None:
        a.ids, a.n_slots, a.n_expert = ids.data_ptr(), ns, n_expert
        a.gate_expert_stride = a.up_expert_stride = B.row_size(t, k) * m
    K.check(K.lib.mi355_glu_matvec(a, _stream()), "mi355_glu_matvec")
    return dst, g, u, oq, ods


_dl_sync = {}


def decode_layer_sync(n_calls=1):
    """A zeroed block of n_calls x mi355_decode_layer_sync_bytes() on the current device (memset on the current stream)."""
    nb = K.lib.mi355_decode_layer_sync_bytes()
    key = (torch.cuda.current_device(), n_calls)
    buf = _dl_sync.get(key)
    if buf is None:
        buf = _dl_sync[key] = torch.empty(n_calls * nb, dtype=torch.uint8, device="cuda")
    buf.zero_()
    return buf, nb


def decode_layer(types, w, n_embd, k_o, n_ff, attn, residual, ffn_norm_w, eps=1e-5, glu_op=2, tail=None, keep=True, sync=None, bufs=None):
    """The persistent decode-layer launch (mi355_decode_layer).  types = (type_o, type_gu, type_d); w = (wo, w_gate, w_up, w_down)
    uint8 block tensors; attn = f32 [k_o] or (act_q, act_ds); tail = None | ("qkv", QkvRopeArgs with everything but norm_x set) |
    ("rows", MmvqArgs with everything but src_f32 set).  bufs: output tensors to use instead of fresh ones, by name (tests place
    them on top of each other the way ggml-alloc does).  -> dict of the f32 outputs (+ "sync": the sync block, error word last)."""
    dev = w[0].device
    bufs = bufs or {}
    f = lambda name, n: bufs[name] if name in bufs else torch.full((n,), float("nan"), dtype=torch.float32, device=dev)
    o = {"ffn_inp": f("ffn_inp", n_embd), "ffn_norm": f("ffn_norm", n_embd), "hidden": f("hidden", n_ff), "l_out": f("l_out", n_embd)}
    if keep:
        o.update({"attn_out": f("attn_out", n_embd), "gate": f("gate", n_ff), "up": f("up", n_ff), "down": f("down", n_embd)})
    a = K.DecodeLayerArgs()
    a.type_o, a.type_gu, a.type_d, a.glu_op = types[0], types[1], types[2], glu_op
    a.n_embd, a.k_o, a.n_ff = n_embd, k_o, n_ff
    a.wo, a.wo_row_stride = _u8(w[0]).data_ptr(), B.row_size(types[0], k_o)
    if isinstance(attn, tuple):
        a.attn_q, a.attn_ds = attn[0].data_ptr(), attn[1].data_ptr()
    else:
        a.attn_f32 = attn.data_ptr()
    a.residual, a.ffn_inp = residual.data_ptr(), o["ffn_inp"].data_ptr()
    a.ffn_norm_w, a.ffn_norm_out, a.norm_eps = ffn_norm_w.data_ptr(), o["ffn_norm"].data_ptr(), eps
    a.w_gate, a.w_up, a.gu_row_stride = _u8(w[1]).data_ptr(), _u8(w[2]).data_ptr(), B.row_size(types[1], n_embd)
    a.hidden = o["hidden"].data_ptr()
    a.w_down, a.down_row_stride = _u8(w[3]).data_ptr(), B.row_size(types[2], n_ff)
    a.l_out = o["l_out"].data_ptr()
    if keep:
        a.attn_out, a.gate_out, a.up_out, a.down_out = (o[n].data_ptr() for n in ("attn_out", "gate", "up", "down"))
    a.tail = K.TAIL_NONE
    if tail is not None and tail[0] == "qkv":
        a.tail, a.qkv = K.TAIL_QKV, tail[1]
        a.qkv.norm_x = o["l_out"].data_ptr()
    elif tail is not None:
        a.tail, a.out = K.TAIL_ROWS, tail[1]
        a.out.src_f32 = o["l_out"].data_ptr()
    if sync is None:
        sync = decode_layer_sync()[0]
    K.check(K.lib.mi355_decode_layer(a, sync.data_ptr(), _stream()), "mi355_decode_layer")
    o["sync"] = sync
    return o


def moe_down_matvec(t, w, m, k, n_expert, aq, ads, ids, weights, residual=None, in_place=False):
    """Fused expert feed-forward output of one decode token (mi355_moe_down_matvec): w = [n_expert][m rows] blocks, aq / ads =
    q8_1 of the [n_slots, k] activations, ids int32 [n_slots], weights f32 [n_slots]
    -> (y [n_slots, m] | None when in_place, weighted [n_slots, m], sum [m], sum + residual [m] | None)."""
    _u8(w)
    ns, dev = ids.numel(), w.device
    y = None if in_place else torch.full((ns, m), float("nan"), dtype=torch.float32, device=dev)
    yw = torch.full((ns, m), float("nan"), dtype=torch.float32, device=dev)
    sm = torch.full((m,), float("nan"), dtype=torch.float32, device=dev)
    ro = torch.full((m,), float("nan"), dtype=torch.float32, device=dev) if residual is not None else None
    a = K.MoeDownArgs()
    a.type, a.n_slots, a.n_expert, a.W = t, ns, n_expert, w.data_ptr()
    a.w_row_stride = B.row_size(t, k)
    a.w_expert_stride = a.w_row_stride * m
    a.m, a.k, a.act_q, a.act_ds, a.ids, a.weights = m, k, aq.data_ptr(), ads.data_ptr(), ids.data_ptr(), weights.data_ptr()
    a.out, a.weighted_out, a.sum_out = None if in_place else y.data_ptr(), yw.data_ptr(), sm.data_ptr()
    if residual is not None:
        a.residual, a.residual_out = residual.data_ptr(), ro.data_ptr()
    K.check(K.lib.mi355_moe_down_matvec(a, _stream()), "mi355_moe_down_matvec")
    return y, yw, sm, ro


def mul_mat_id_dq(t, as_, b, ids, m, n_expert):
    """ggml_mul_mat_id for prefill-sized batches (device-side expert bucketing + one bf16-MFMA GEMM launch):
    as_ = [n_expert][m rows] blocks, b = [n_tokens, b_ne1, k] f32, ids = [n_tokens, n_used] int32 -> [n_tokens, n_used, m] f32."""
    _u8(as_)
    assert b.dim() == 3 and b.is_contiguous() and ids.dtype == torch.int32 and ids.dim() == 2 and ids.is_contiguous()
    n_tok, b_ne1, k = b.shape
    n_used = ids.shape[1]
    rs = B.row_size(t, k)
    need = K.lib.mi355_mul_mat_id_dq_workspace_bytes(k, n_tok, b_ne1, n_used, n_expert)
    ws = torch.empty(need, dtype=torch.uint8, device=b.device)
    dst = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device)
    K.check(K.lib.mi355_mul_mat_id_dq(t, as_.data_ptr(), rs, rs * m, b.data_ptr(), k * 4, b_ne1 * k * 4, ids.data_ptr(), n_used,
                                      dst.data_ptr(), m, k, n_expert, n_used, n_tok, b_ne1, ws.data_ptr(), need, _stream()),
            "mi355_mul_mat_id_dq")
    return dst


def mul_mat_id_skinny(t, as_, b, ids, m, n_expert):
    """ggml_mul_mat_id for small batches (device-side bucketing + skinny int8-MFMA kernels, every expert streamed once
    per 32 of its columns); same arguments and result layout as mul_mat_id_dq."""
    _u8(as_)
    assert b.dim() == 3 and b.is_contiguous() and ids.dtype == torch.int32 and ids.dim() == 2 and ids.is_contiguous()
    n_tok, b_ne1, k = b.shape
    n_used = ids.shape[1]
    rs = B.row_size(t, k)
    need = K.lib.mi355_mul_mat_id_skinny_workspace_bytes(t, k, n_tok, b_ne1, n_used, n_expert)
    ws = torch.empty(need, dtype=torch.uint8, device=b.device)
    dst = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device)
    K.check(K.lib.mi355_mul_mat_id_skinny(t, as_.data_ptr(), rs, rs * m, b.data_ptr(), k * 4, b_ne1 * k * 4, ids.data_ptr(), n_used,
                                          dst.data_ptr(), m, k, n_expert, n_used, n_tok, b_ne1, ws.data_ptr(), need, _stream()),
            "mi355_mul_mat_id_skinny")
    return dst


def mul_mat_id_skinny_pair(t, as0, as1, b, ids, m, n_expert):
    """two expert tensors (ffn_up_exps, ffn_gate_exps) on the same b and ids in one skinny launch -> two [n_tokens, n_used, m]."""
    _u8(as0); _u8(as1)
    n_tok, b_ne1, k = b.shape
    n_used = ids.shape[1]
    rs = B.row_size(t, k)
    need = K.lib.mi355_mul_mat_id_skinny_workspace_bytes(t, k, n_tok, b_ne1, n_used, n_expert)
    ws = torch.empty(need, dtype=torch.uint8, device=b.device)
    d0 = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device)
    d1 = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device)
    K.check(K.lib.mi355_mul_mat_id_skinny_pair(t, as0.data_ptr(), as1.data_ptr(), rs, rs * m, b.data_ptr(), k * 4, b_ne1 * k * 4, ids.data_ptr(),
                                               n_used, d0.data_ptr(), d1.data_ptr(), m, k, n_expert, n_used, n_tok, b_ne1, ws.data_ptr(), need,
                                               _stream()), "mi355_mul_mat_id_skinny_pair")
    return d0, d1


def mul_mat_id_skinny_ex(t, as0, as1, b, ids, m, n_expert, ws, tables, flags):
    """mi355_mul_mat_id_skinny_ex on a caller-kept workspace and routing-table buffer (flags: 1 = the workspace already holds b's
    activation planes, 2 = `tables` already holds the tables of these ids); as1 None: one tensor -> dst0 (, dst1)."""
    n_tok, b_ne1, k = b.shape
    n_used = ids.shape[1]
    rs = B.row_size(t, k)
    d0 = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device)
    d1 = torch.full((n_tok, n_used, m), float("nan"), dtype=torch.float32, device=b.device) if as1 is not None else None
    K.check(K.lib.mi355_mul_mat_id_skinny_ex(t, as0.data_ptr(), as1.data_ptr() if as1 is not None else None, rs, rs * m, b.data_ptr(), k * 4,
                                             b_ne1 * k * 4, ids.data_ptr(), n_used, d0.data_ptr(), d1.data_ptr() if d1 is not None else None, m, k,
                                             n_expert, n_used, n_tok, b_ne1, ws.data_ptr(), ws.numel(), tables.data_ptr() if tables is not None else None,
                                             flags, _stream()), "mi355_mul_mat_id_skinny_ex")
    return (d0, d1) if as1 is not None else d0


def mul_mat_skinny(t, w, b, m):
    """MUL_MAT for small batches through the int8-MFMA skinny kernel, in passes of 32 columns: b = [n, k] f32 -> [n, m]."""
    _u8(w)
    n, k = b.shape
    aq, ads = quantize_act(b)
    dst = torch.empty((n, m), dtype=torch.float32, device=b.device)
    for c0 in range(0, n, 32):
        nc = min(32, n - c0)
        K.check(K.lib.mi355_mul_mat_skinny(t, w.data_ptr(), B.row_size(t, k), aq[c0:].data_ptr(), ads[c0:].data_ptr(),
                                           dst[c0:].data_ptr(), m, m, k, nc, _stream()), "mi355_mul_mat_skinny")
    return dst


def quantize_act_q8k(x):
    """[n, k] f32 -> q8_K planes (int8 [n, k], f32 [n, k/256], int16 [n, k/16])."""
    n, k = x.shape
    q = torch.empty((n, k), dtype=torch.int8, device=x.device)
    d = torch.empty((n, k // 256), dtype=torch.float32, device=x.device)
    bs = torch.empty((n, k // 16), dtype=torch.int16, device=x.device)
    K.check(K.lib.mi355_quantize_act_q8k(x.data_ptr(), q.data_ptr(), d.data_ptr(), bs.data_ptr(), k, n, 1, 1, x.stride(0) * 4, 0, 0, _stream()),
            "mi355_quantize_act_q8k")
    return q, d, bs


def mul_mat_skinny_k(t, w, b, m, pass_cols=32):
    """K-quant MUL_MAT on q8_K activations through the digit-split int8-MFMA kernel, passes of 32 (or 64: two column tiles per
    workgroup) columns."""
    _u8(w)
    n, k = b.shape
    q, d, bs = quantize_act_q8k(b)
    dst = torch.empty((n, m), dtype=torch.float32, device=b.device)
    for c0 in range(0, n, pass_cols):
        K.check(K.lib.mi355_mul_mat_skinny_k(t, w.data_ptr(), B.row_size(t, k), q[c0:].data_ptr(), d[c0:].data_ptr(), bs[c0:].data_ptr(),
                                             dst[c0:].data_ptr(), m, m, k, min(pass_cols, n - c0), _stream()), "mi355_mul_mat_skinny_k")
    return dst


def mul_mat_skinny_k_group(t, ws, b, ms):
    """Up to four K-quant matrices of type t against the same [n <= 64, k] activations in one launch -> list of [n, m_i]."""
    import ctypes as C
    n, k = b.shape
    q, d, bs = quantize_act_q8k(b)
    cnt = len(ws)
    dsts = [torch.empty((n, m), dtype=torch.float32, device=b.device) for m in ms]
    Wp = (C.c_void_p * cnt)(*[_u8(w).data_ptr() for w in ws])
    rs = (C.c_int64 * cnt)(*[B.row_size(t, k)] * cnt)
    dp = (C.c_void_p * cnt)(*[x.data_ptr() for x in dsts])
    mm = (C.c_int64 * cnt)(*ms)
    K.check(K.lib.mi355_mul_mat_skinny_k_group(t, cnt, Wp, rs, dp, mm, mm, q.data_ptr(), d.data_ptr(), bs.data_ptr(), k, n, _stream()),
            "mi355_mul_mat_skinny_k_group")
    return dsts


def mul_mat_qk(t, w, b, m):
    """K-quant prefill MUL_MAT on q8_K activations (digit-split int8-MFMA tile kernel): b = [n, k] f32 -> [n, m]."""
    _u8(w)
    n, k = b.shape
    q, d, bs = quantize_act_q8k(b)
    dst = torch.empty((n, m), dtype=torch.float32, device=b.device)
    K.check(K.lib.mi355_mul_mat_qk(t, w.data_ptr(), B.row_size(t, k), q.data_ptr(), d.data_ptr(), bs.data_ptr(), dst.data_ptr(), m, m, k, n,
                                   _stream()), "mi355_mul_mat_qk")
    return dst


def _desc(t, type_id):
    """ggml-style descriptor of a torch tensor of up to 4 dims (last dim fastest), strides honoured"""
    d = K.Tensor()
    d.data, d.type = t.data_ptr(), type_id
    shape, stride = list(t.shape)[::-1], list(t.stride())[::-1]
    es = t.element_size()
    for i in range(4):
        d.ne[i] = shape[i] if i < len(shape) else 1
        d.nb[i] = stride[i] * es if i < len(shape) else (d.nb[i - 1] * d.ne[i - 1] if i else es)
    return d


def mul_mat_f(type_a, a, b, type_b=B.F32):
    """MUL_MAT on float weights (mi355_mul_mat_f): a [.., m, k] (f32 | f16 | bf16 bits as a torch tensor of matching width),
    b [.., n, k] f32 | f16 -> [.., n, m] f32; leading dims broadcast ggml-style."""
    assert a.is_cuda and b.is_cuda
    lead = list(b.shape[:-2])
    dst = torch.empty(lead + [b.shape[-2], a.shape[-2]], dtype=torch.float32, device=b.device)
    ta, tb, td = _desc(a, type_a), _desc(b, type_b), _desc(dst, B.F32)
    K.check(K.lib.mi355_mul_mat_f(ta, tb, td, _stream()), "mi355_mul_mat_f")
    return dst


def get_rows(t, w, ids, k):
    """GGML_OP_GET_ROWS (mi355_get_rows): w uint8 [nrows, row_bytes] blocks of type t (k values per row), ids int32 [n] or
    [b, n] -> f32 [.., n, k], row ids[.., i] dequantized."""
    assert w.is_cuda and ids.is_cuda and ids.dtype == torch.int32 and w.dtype == torch.uint8 and w.dim() == 2
    dst = torch.empty(list(ids.shape) + [k], dtype=torch.float32, device=w.device)
    ts = K.Tensor()
    ts.data, ts.type = w.data_ptr(), t
    ts.ne[0], ts.ne[1], ts.ne[2], ts.ne[3] = k, w.shape[0], 1, 1
    ts.nb[0], ts.nb[1] = B.TYPE_SIZE[t], w.stride(0)
    ts.nb[2] = ts.nb[3] = 0 if ids.dim() > 1 else w.stride(0) * w.shape[0]     # one table for every batch of ids
    K.check(K.lib.mi355_get_rows(ts, _desc(ids, B.I32), _desc(dst, B.F32), _stream()), "mi355_get_rows")
    return dst


def set_rows(src, ids, dst, type_dst):
    """GGML_OP_SET_ROWS (mi355_set_rows): src f32 [.., n, k], ids int64 [.., n], dst rows of type_dst (f32 / f16 tensors,
    or uint8 rows of q8_0 blocks); writes into dst and returns it."""
    ts, ti = _desc(src, B.F32), _desc(ids, B.I64)
    td = _desc(dst, type_dst)
    if type_dst in (B.Q8_0, B.Q4_0):  # uint8 rows of 34- / 18-byte blocks: extents in elements, nb[0] the block size
        td.ne[0] = dst.shape[-1] // B.TYPE_SIZE[type_dst] * 32
        td.nb[0] = B.TYPE_SIZE[type_dst]
    K.check(K.lib.mi355_set_rows(ts, ti, td, _stream()), "mi355_set_rows")
    return dst


_KV_DTYPE = {B.F32: torch.float32, B.F16: torch.float16, B.BF16: torch.bfloat16, B.Q8_0: torch.uint8, B.Q4_0: torch.uint8}
_KV_BYTES = {B.F32: 4, B.F16: 2, B.BF16: 2, B.Q8_0: 1, B.Q4_0: 1}          # of a cache tensor's element
_BLOCK = {B.Q8_0: 34, B.Q4_0: 18}
_MASK_DTYPE = (torch.float16, torch.int16, torch.uint16)                    # f16 or its bits


# The entry points of the bounded KV cache are called once per layer and step: their wrappers read every tensor's shape and strides once.
# A tensor has to lie on the current device, whose current stream the launch goes to.

# torch.cuda.current_stream(dev).cuda_stream without the Stream object around it (2.7 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _on(dev, *ts):
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensor on {t.device}, the current device is cuda:{dev}")


def _cache_rows(t, type_kv, name, S, hk, slots=None):
    """(slots, values per row, strides) of a cache tensor [seqs, kv heads, slots, row]: f32 / f16 / bf16 values, or uint8 bytes of q8_0 / q4_0
    blocks, contiguous rows"""
    s0, s1, s2, s3 = t.shape
    st = t.stride()
    if t.dtype is not _KV_DTYPE.get(type_kv) or (s3 > 1 and st[3] != 1) or s0 != S or s1 != hk or (slots is not None and s2 != slots):
        raise ValueError(f"{name}: expected [{S} seqs, {hk} kv heads, {'slots' if slots is None else slots}, row] of type {B.TYPE_NAMES.get(type_kv, type_kv)} "
                         f"(f32, f16, bf16, or uint8 bytes of q8_0 / q4_0 blocks), rows contiguous; got {tuple(t.shape)} of {t.dtype}")
    return s2, (s3 // _BLOCK[type_kv] * 32 if type_kv in _BLOCK else s3), st


def qk_norm_rope(q, k, v, q_norm, k_norm, eps, pos, k_cache, v_cache, type_kv, rows=None, slot_pos=None, slot_mass=None, n_dims=None, mode=2,
                 n_ctx_orig=8192, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
                 freq_factors=None, q_out=None):
    """Per-head RMS norm x weight and rotation of q and k, k and v into their cache rows (mi355_qk_norm_rope).  q [seqs, tokens, heads, d],
    k [seqs, tokens, kv heads, d], v [.., dv] (or None, with v_cache None) f32, strides free (contiguous rows); q_norm / k_norm f32 [d] or
    None; pos int32 [seqs, tokens]; caches [seqs, kv heads, slots, row] of type_kv; rows int32 [seqs, kv heads, tokens] (None: token i goes
    to slot i); slot_pos int32, slot_mass f32 [seqs, kv heads, slots] or None -> q rotated, f32 [seqs, heads, tokens, d] (q_out's strides)."""
    f32, i32 = torch.float32, torch.int32
    dev = torch.cuda.current_device()
    _on(dev, q, k, v, q_norm, k_norm, pos, k_cache, v_cache, rows, slot_pos, slot_mass, freq_factors, q_out)
    S, n, H, d = q.shape
    kS, kn, hk, kd = k.shape
    qs, ks = q.stride(), k.stride()
    if q.dtype is not f32 or k.dtype is not f32 or kS != S or kn != n or kd != d or qs[3] != 1 or ks[3] != 1:
        raise ValueError("q and k: f32 [seqs, tokens, heads, d] with contiguous rows")
    if (v is None) != (v_cache is None):
        raise ValueError("v and v_cache come together")
    slots, kd, kc = _cache_rows(k_cache, type_kv, "k_cache", S, hk)
    if kd != d:
        raise ValueError("k_cache: rows of another length than k's")
    eb = _KV_BYTES[type_kv]
    dv, vp, vs, vcp, vc = 0, None, (0, 0, 0, 0), None, (0, 0, 0, 0)
    if v is not None:
        vS, vn, vh, dv = v.shape
        vs = v.stride()
        if v.dtype is not f32 or vS != S or vn != n or vh != hk or vs[3] != 1:
            raise ValueError("v: f32 [seqs, tokens, kv heads, dv] with contiguous rows")
        _, vd, vc = _cache_rows(v_cache, type_kv, "v_cache", S, hk, slots)
        if vd != dv:
            raise ValueError("v_cache: rows of another length than v's")
        vp, vcp = v.data_ptr(), v_cache.data_ptr()
    ps = pos.stride()
    if pos.dtype is not i32 or pos.shape != (S, n):
        raise ValueError("pos: int32 [seqs, tokens]")
    rp, rs = None, (0, 0, 0)
    if rows is not None:
        if rows.dtype is not i32 or rows.shape != (S, hk, n):
            raise ValueError("rows: int32 [seqs, kv heads, tokens]")
        rp, rs = rows.data_ptr(), rows.stride()
    spp, sps, smp, sms = None, (0, 0, 0), None, (0, 0, 0)
    if slot_pos is not None:
        spp, sps = slot_pos.data_ptr(), slot_pos.stride()
        if slot_pos.dtype is not i32 or slot_pos.shape != (S, hk, slots) or (slots > 1 and sps[2] != 1):
            raise ValueError("slot_pos: int32 [seqs, kv heads, slots], slots contiguous")
    if slot_mass is not None:
        smp, sms = slot_mass.data_ptr(), slot_mass.stride()
        if slot_mass.dtype is not f32 or slot_mass.shape != (S, hk, slots) or (slots > 1 and sms[2] != 1):
            raise ValueError("slot_mass: f32 [seqs, kv heads, slots], slots contiguous")
    n_dims = d if n_dims is None else n_dims
    for t, m in ((q_norm, d), (k_norm, d), (freq_factors, n_dims // 2)):
        if t is not None and (t.dtype is not f32 or t.numel() < m or not t.is_contiguous()):
            raise ValueError("q_norm, k_norm: f32 [d]; freq_factors: f32 [n_dims / 2]")
    if q_out is None:
        q_out = torch.empty((S, H, n, d), dtype=f32, device=q.device)
    elif q_out.dtype is not f32 or q_out.shape != (S, H, n, d) or q_out.stride(3) != 1:
        raise ValueError("q_out: f32 [seqs, heads, tokens, d] with contiguous rows")
    if S == 0 or n == 0:
        return q_out
    os = q_out.stride()
    a = K.QkNormRopeArgs(
        q.data_ptr(), qs[1] * 4, qs[2] * 4, qs[0] * 4, k.data_ptr(), ks[1] * 4, ks[2] * 4, ks[0] * 4, vp, vs[1] * 4, vs[2] * 4, vs[0] * 4,
        q_norm.data_ptr() if q_norm is not None else None, k_norm.data_ptr() if k_norm is not None else None,
        q_out.data_ptr(), os[2] * 4, os[1] * 4, os[0] * 4, k_cache.data_ptr(), kc[2] * eb, kc[1] * eb, kc[0] * eb, vcp, vc[2] * eb, vc[1] * eb, vc[0] * eb,
        rp, rs[2] * 4, rs[1] * 4, rs[0] * 4, pos.data_ptr(), ps[1] * 4, ps[0] * 4, freq_factors.data_ptr() if freq_factors is not None else None,
        spp, sps[1] * 4, sps[0] * 4, smp, sms[1] * 4, sms[0] * 4, d, dv, H, hk, n, S, slots,
        type_kv, n_dims, mode, n_ctx_orig, eps, freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow)
    rc = K.lib.mi355_qk_norm_rope(a, _raw_stream(dev))
    if rc:
        raise K.Mi355Error(rc, "mi355_qk_norm_rope")
    return q_out


def kv_evict(mass, slot_pos, n_past, n_keep, n_sink=0, n_recent=0, n_used=None, n_evict=None, k=None, v=None, type_kv=B.F16, d=None, k_out=None, v_out=None):
    """The slots to keep (mi355_kv_evict): mass f32, slot_pos int32 [seqs, kv heads, slots] (slots contiguous), n_past / n_used int32 [seqs]
    -> (kept int32 [seqs, kv heads, n_keep], evicted int32 [.., n_evict]); n_evict None: slots - n_keep.  With caches k, v [seqs, kv heads,
    slots, row] of type_kv their kept rows are gathered too, into k_out, v_out [seqs, kv heads, n_keep, row] (None: new)
    -> (kept, evicted, mass of the kept, positions of the kept), or (.., k_out, v_out) where those were None."""
    i32 = torch.int32
    dev = torch.cuda.current_device()
    _on(dev, mass, slot_pos, n_past, n_used, k, v, k_out, v_out)
    S, hk, slots = mass.shape
    ms, ps = mass.stride(), slot_pos.stride()
    if mass.dtype is not torch.float32 or slot_pos.dtype is not i32 or slot_pos.shape != (S, hk, slots) or (slots > 1 and (ms[2] != 1 or ps[2] != 1)):
        raise ValueError("mass f32, slot_pos int32: [seqs, kv heads, slots], slots contiguous")
    for t in (n_past, n_used):
        if t is not None and (t.dtype is not i32 or t.shape != (S,) or (S > 1 and t.stride(0) != 1)):
            raise ValueError("n_past, n_used: int32 [seqs]")
    if (k is None) != (v is None) or (k_out is None) != (v_out is None) or (k is None and k_out is not None):
        raise ValueError("k and v, and k_out and v_out, come together")
    n_evict = max(0, slots - n_keep) if n_evict is None else n_evict
    keep, ev = max(n_keep, 0), max(n_evict, 0)
    kept = torch.empty((S, hk, keep), dtype=i32, device=mass.device)
    evicted = torch.empty((S, hk, ev), dtype=i32, device=mass.device)
    rows, tables, ret = (None, 0, 0, 0) * 4, (None, 0, 0) * 2, (kept, evicted)
    dk = dv = 0
    if k is not None:
        _, dk, ks = _cache_rows(k, type_kv, "k", S, hk, slots)
        _, dv, vs = _cache_rows(v, type_kv, "v", S, hk, slots)
        if d is not None and d != dk:
            raise ValueError(f"k: rows of {dk} values, not {d}")
        new = k_out is None
        if new:
            k_out, v_out = (torch.zeros((S, hk, keep, t.shape[3]), dtype=t.dtype, device=t.device) for t in (k, v))
        _, ko, kos = _cache_rows(k_out, type_kv, "k_out", S, hk, n_keep)
        _, vo, vos = _cache_rows(v_out, type_kv, "v_out", S, hk, n_keep)
        if ko != dk or vo != dv:
            raise ValueError("k_out, v_out: rows of another length than k's, v's")
        b = _KV_BYTES[type_kv]
        mass_out = torch.empty((S, hk, keep), dtype=torch.float32, device=mass.device)
        pos_out = torch.empty((S, hk, keep), dtype=i32, device=mass.device)
        rows = (k.data_ptr(), ks[2] * b, ks[1] * b, ks[0] * b, v.data_ptr(), vs[2] * b, vs[1] * b, vs[0] * b,
                k_out.data_ptr(), kos[2] * b, kos[1] * b, kos[0] * b, v_out.data_ptr(), vos[2] * b, vos[1] * b, vos[0] * b)
        tables = (mass_out.data_ptr(), keep * 4, hk * keep * 4, pos_out.data_ptr(), keep * 4, hk * keep * 4)
        ret = (kept, evicted, mass_out, pos_out, k_out, v_out) if new else (kept, evicted, mass_out, pos_out)
    a = K.KvEvictArgs(mass.data_ptr(), ms[1] * 4, ms[0] * 4, slot_pos.data_ptr(), ps[1] * 4, ps[0] * 4,
                      n_used.data_ptr() if n_used is not None else None, n_past.data_ptr(), kept.data_ptr(), keep * 4, hk * keep * 4,
                      evicted.data_ptr() if ev else None, ev * 4, hk * ev * 4, *rows, *tables, slots, n_keep, n_evict, hk, S, dk, dv, type_kv, n_sink, n_recent)
    rc = K.lib.mi355_kv_evict(a, _raw_stream(dev))
    if rc:
        raise K.Mi355Error(rc, "mi355_kv_evict")
    return ret


def _mass_args(dev, q, k, v, mask, type_kv, scale, mass, decay, mass_out, max_bias, logit_softcap):
    """checks and arguments that flash_attn_ext_mass and attn_mass (v None) share -> (FattnArgs, AttnMassArgs, dst | None, mass_out)"""
    f32 = torch.float32
    _on(dev, q, k, v, mask, mass, mass_out)
    S, H, n, d = q.shape
    qs = q.stride()
    if q.dtype is not f32 or qs[3] != 1:
        raise ValueError("q: f32 [seqs, heads, tokens, d] with contiguous rows")
    hk = k.shape[1]
    slots, kd, ks = _cache_rows(k, type_kv, "k", S, hk)
    if kd != d:
        raise ValueError("k: rows of another length than q's")
    b = _KV_BYTES[type_kv]
    mp, m1, m2, m3, e2, e3 = None, 0, 0, 0, 0, 0
    if mask is not None:
        sh, st = mask.shape, mask.stride()
        if len(sh) < 4:                       # the two first dimensions may be left out, or the heads'
            sh, st = ((1, 1) + sh, (0, 0) + st) if len(sh) == 2 else ((sh[0], 1) + sh[1:], (st[0], 0) + st[1:])
        e3, e2, m_n, m_s = sh
        if (mask.dtype is not torch.float16 and mask.dtype not in _MASK_DTYPE) or e2 < 1 or e3 < 1 or H % e2 or S % e3 or m_n < n or m_s != slots or (slots > 1 and st[3] != 1):
            raise ValueError("mask: f16 (or its bits as int16 / uint16) [seqs | 1, heads | 1, >= tokens, slots], the two first may be left out")
        mp, m1, m2, m3 = mask.data_ptr(), st[2] * 2, st[1] * 2, st[0] * 2
    dst, vp, v1, v2, v3, dp, dv = None, None, 0, 0, 0, None, 0
    if v is not None:
        _, dv, vs = _cache_rows(v, type_kv, "v", S, hk, slots)
        dst = torch.empty((S, n, H, dv), dtype=f32, device=q.device)
        vp, v1, v2, v3, dp = v.data_ptr(), vs[2] * b, vs[1] * b, vs[0] * b, dst.data_ptr()
    if mass_out is None:
        mass_out = torch.empty((S, hk, slots), dtype=f32, device=q.device)
        os = (hk * slots, slots, 1)
    else:
        os = mass_out.stride()
        if mass_out.dtype is not f32 or mass_out.shape != (S, hk, slots) or (slots > 1 and os[2] != 1):
            raise ValueError("mass_out: f32 [seqs, kv heads, slots], slots contiguous")
    ip, ns = None, (0, 0, 0)
    if mass is not None:
        ip, ns = mass.data_ptr(), mass.stride()
        if mass.dtype is not f32 or mass.shape != (S, hk, slots) or (slots > 1 and ns[2] != 1):
            raise ValueError("mass: f32 [seqs, kv heads, slots], slots contiguous")
    if n == 0 or S == 0:
        return None, None, dst, mass_out
    a = K.FattnArgs(q.data_ptr(), qs[2] * 4, qs[1] * 4, qs[0] * 4, k.data_ptr(), type_kv, ks[2] * b, ks[1] * b, ks[0] * b, vp, type_kv, v1, v2, v3,
                    mp, m1, m2, m3, e2, e3, dp, dv * 4, H * dv * 4, n * H * dv * 4, d, n, slots, H, hk, S, scale, max_bias, logit_softcap, dv)
    return a, K.AttnMassArgs(ip, ns[1] * 4, ns[0] * 4, mass_out.data_ptr(), os[1] * 4, os[0] * 4, decay), dst, mass_out


def _no_queries(mass, decay, mass_out):
    """mass_out of a call without queries: what the earlier ones left"""
    return mass_out.zero_() if mass is None or decay == 0.0 else torch.mul(mass, decay, out=mass_out)


def flash_attn_ext_mass(q, k, v, mask, type_kv, scale, mass=None, decay=1.0, mass_out=None, max_bias=0.0, logit_softcap=0.0):
    """A decode step's attention and the weight every slot draws (mi355_flash_attn_ext_mass).  q f32 [seqs, heads, tokens <= 8, d], k, v
    [seqs, kv heads, slots, row] of type_kv, mask f16 [seqs | 1, heads | 1, >= tokens, slots] (or [seqs | 1, tokens, slots], [tokens, slots],
    None); mass f32 [seqs, kv heads, slots] or None; mass_out may be mass -> (f32 [seqs, tokens, heads, dv], mass_out = decay mass + weights)."""
    dev = torch.cuda.current_device()
    a, w, dst, mass_out = _mass_args(dev, q, k, v, mask, type_kv, scale, mass, decay, mass_out, max_bias, logit_softcap)
    if a is None:
        return dst, _no_queries(mass, decay, mass_out)
    need = K.lib.mi355_flash_attn_ext_mass_workspace_bytes(a)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    rc = K.lib.mi355_flash_attn_ext_mass(a, w, ws.data_ptr(), need, _raw_stream(dev))
    if rc:
        raise K.Mi355Error(rc, "mi355_flash_attn_ext_mass")
    return dst, mass_out


def attn_mass(q, k, mask, type_kv, scale, mass=None, decay=1.0, mass_out=None, max_bias=0.0, logit_softcap=0.0):
    """The weight every slot draws from up to 65535 queries (mi355_attn_mass); arguments as flash_attn_ext_mass, without V -> mass_out."""
    dev = torch.cuda.current_device()
    a, w, _, mass_out = _mass_args(dev, q, k, None, mask, type_kv, scale, mass, decay, mass_out, max_bias, logit_softcap)
    if a is None:
        return _no_queries(mass, decay, mass_out)
    need = K.lib.mi355_attn_mass_workspace_bytes(a)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    rc = K.lib.mi355_attn_mass(a, w, ws.data_ptr(), need, _raw_stream(dev))
    if rc:
        raise K.Mi355Error(rc, "mi355_attn_mass")
    return mass_out
