// qk_norm_rope.hip -- attention input of models that normalise queries and keys per head: RMS norm x weight and the position rotation of
// every q and k head, and the store of k and v into their cache rows, in one launch (mi355_qk_norm_rope).
//
//   y = x / sqrt(mean(x^2) + eps) * w            over a head's head_dim values
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = pos * f_i,  pairs (2i, 2i + 1) NORMAL, (i, i + n_dims / 2) NEOX
// Angles are formed and reduced to one turn in 64 bits: in 32 bits the product alone is off by 0.01 rad at position 10^5.
#include "row_formats.h"
#include "rope.h"
#include "spans.h"

namespace {

struct QnArgs {
    const char * q, * k, * v;
    int64_t q_nb1, q_nb2, q_nb3, k_nb1, k_nb2, k_nb3, v_nb1, v_nb2, v_nb3;
    const float * qw, * kw, * ff;
    char * qo, * ko, * vo;
    int64_t qo_nb1, qo_nb2, qo_nb3, ko_nb1, ko_nb2, ko_nb3, vo_nb1, vo_nb2, vo_nb3;
    const char * pos, * rows;
    int64_t pos_nb1, pos_nb3, rows_nb1, rows_nb2, rows_nb3;
    char * slot_pos, * slot_mass;
    int64_t sp_nb2, sp_nb3, sm_nb2, sm_nb3;
    int64_t n_rows;
    double log2_step;           // pair i turns by 2^(-i log2_step) / (2 pi) revolutions per position (before YaRN and freq_factors)
    float eps, mscale, freq_scale, ext_factor, corr0, corr1;
    int d, dv, n_dims, neox, n_head, n_head_kv, n, ne3;
};

// revolutions per position of pair i
static __device__ __forceinline__ double qn_freq(const QnArgs & a, int i) {
    double w = exp2(-(double)i * a.log2_step) * 0.15915494309189533577;
    if (a.ff) w /= (double)a.ff[i];
    double f = (double)a.freq_scale;
    if (a.ext_factor != 0.0f) {                       // YaRN: interpolated and extrapolated angle mixed by a ramp over the pairs
        const float y = (i - a.corr0) / fmaxf(0.001f, a.corr1 - a.corr0);
        const float mix = (1.0f - fminf(1.0f, fmaxf(0.0f, y))) * a.ext_factor;
        f = f * (1.0 - (double)mix) + (double)mix;
    }
    return w * f;
}

// 4 consecutive values of a row
template <int TYPE> static __device__ __forceinline__ void qn_store4(char * row, int e, const float * v) {
    if (TYPE == MI355_TYPE_F32) *(v4f *)((float *)row + e) = v4f{v[0], v[1], v[2], v[3]};
    else {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = TYPE == MI355_TYPE_F16 ? __half_as_ushort(cvt<float, __half>(v[i])) : cvt<float, bf16_bits>(v[i]).bits;
        *(v2i *)((uint16_t *)row + e) = v2i{h[0] | h[1] << 16, h[2] | h[3] << 16};
    }
}

// A group of L lanes takes a row (a head of q, k or v of one token), 8 values a lane: rotating rows as 4 and 4 values whose pairs the lane
// holds itself -- NEOX: 4 i.. and n_dims / 2 + 4 i..; NORMAL and the features past n_dims: 8 i.. -- so nothing crosses lanes but the sum of
// squares.  A workgroup first forms cos and sin of all pairs of its TT tokens in LDS (64-bit angles: ~100 clocks a pair, shared by every head),
// then walks their rows two at a time, loads ahead.  Bound by the rows' bytes at prompts (8192 tokens x 64 / 8 heads of 128 in f16:
// 638 MB in 138-149 us, 4.3-4.6 TB/s, into q8_0 or q4_0 caches 147 for the whole call; 1111 tokens x 24 / 4 heads of 96 in bf16: 10.6 us), by one launch
// at steps (4.3 us, 6.0 with blocks to quantize: 16 sequences x 64 / 8 heads, a quarter of a row's lanes take 32 values each).
constexpr int QN_THREADS = 256;

template <int TYPE, int L>
__global__ void __launch_bounds__(QN_THREADS)
qk_norm_rope_kernel(const QnArgs a, int tt, int chunks) {
    constexpr bool quant = TYPE == MI355_TYPE_Q8_0 || TYPE == MI355_TYPE_Q4_0;
    constexpr int G = QN_THREADS / L;
    extern __shared__ __attribute__((aligned(16))) float cs[];       // [tt][2][n_dims / 2], then rows to quantize [G][8 L]
    const int tid = threadIdx.x, j = tid % L, g = tid / L, half = a.n_dims / 2;
    const int t0 = blockIdx.x / chunks * tt, chunk = blockIdx.x % chunks, T = a.n * a.ne3, nt = T - t0 < tt ? T - t0 : tt;
    const int H = a.n_head, HK = a.n_head_kv, R = H + (a.vo ? 2 : 1) * HK;

    const bool rotates = 8 * j < a.n_dims, in = 8 * j < a.d, vin = 8 * j < a.dv;
    const int ea = a.neox && rotates ? 4 * j : 8 * j, eb = a.neox && rotates ? half + 4 * j : 8 * j + 4;
    // rows of this workgroup's chunk: (token, row) pairs n = chunk * G + g, + chunks * G, ...
    struct Row { const float * src; int t, i3, r, kind; };            // kind: 0 q, 1 k, 2 v
    auto locate = [&](int n) {
        Row x;
        const int tok = t0 + n / R;
        x.r = n % R;
        x.i3 = tok / a.n; x.t = tok - x.i3 * a.n;
        x.kind = x.r < H ? 0 : x.r < H + HK ? 1 : 2;
        if (x.kind) x.r -= x.kind == 1 ? H : H + HK;
        x.src = (const float *)(x.kind == 0 ? a.q + x.t * a.q_nb1 + x.r * a.q_nb2 + x.i3 * a.q_nb3 : x.kind == 1 ? a.k + x.t * a.k_nb1 + x.r * a.k_nb2 + x.i3 * a.k_nb3
                                                                                                                : a.v + x.t * a.v_nb1 + x.r * a.v_nb2 + x.i3 * a.v_nb3);
        return x;
    };
    auto load = [&](const Row & x, v4f & A, v4f & B) {
        A = B = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (x.kind == 2 ? vin : in) { A = *(const v4f *)(x.src + (x.kind == 2 ? 8 * j : ea)); B = *(const v4f *)(x.src + (x.kind == 2 ? 8 * j + 4 : eb)); }
    };
    const int rows = nt * R, step = chunks * G;
    int n = chunk * G + g;
    Row x0, x1;
    v4f A0, B0, A1, B1;
    if (n < rows) { x0 = locate(n); load(x0, A0, B0); }
    if (n + step < rows) { x1 = locate(n + step); load(x1, A1, B1); }

    for (int i = tid; i < nt * half; i += QN_THREADS) {
        const int tok = i / half, p = i - tok * half, i3 = (t0 + tok) / a.n, t = t0 + tok - i3 * a.n;
        const double rev = (double)*(const int32_t *)(a.pos + t * a.pos_nb1 + i3 * a.pos_nb3) * qn_freq(a, p);
        float c, s;
        sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
        cs[tok * 2 * half + p] = c * a.mscale;
        cs[tok * 2 * half + half + p] = s * a.mscale;
    }
    v4f wq[2], wk[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        wq[i] = wk[i] = v4f{1.0f, 1.0f, 1.0f, 1.0f};
        if (in && a.qw) wq[i] = *(const v4f *)(a.qw + (i ? eb : ea));
        if (in && a.kw) wk[i] = *(const v4f *)(a.kw + (i ? eb : ea));
    }
    __syncthreads();

    while (n < rows) {
        const Row x = x0;
        float A[4] = {A0[0], A0[1], A0[2], A0[3]}, B[4] = {B0[0], B0[1], B0[2], B0[3]};
        const int tok = n / R;
        x0 = x1; A0 = A1; B0 = B1;
        if (n + 2 * step < rows) { x1 = locate(n + 2 * step); load(x1, A1, B1); }
        n += step;
        if (x.kind != 2) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) ss += A[i] * A[i];
#pragma unroll
            for (int i = 0; i < 4; i++) ss += B[i] * B[i];
            ss += dpp_f32<0xB1>(ss);
            ss += dpp_f32<0x4E>(ss);
            ss += dpp_f32<0x141>(ss);
            if (L >= 16) ss += dpp_f32<0x140>(ss);
            if (L == 32) ss += __shfl_xor(ss, 16, 64);
            const float s = 1.0f / sqrtf(ss / a.d + a.eps);
            const v4f w0 = x.kind == 0 ? wq[0] : wk[0], w1 = x.kind == 0 ? wq[1] : wk[1];
#pragma unroll
            for (int i = 0; i < 4; i++) { A[i] = A[i] * s * w0[i]; B[i] = B[i] * s * w1[i]; }
            if (rotates) {
                const v4f c = *(const v4f *)(cs + tok * 2 * half + 4 * j), sn = *(const v4f *)(cs + tok * 2 * half + half + 4 * j);
                if (a.neox) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float u = A[i], v = B[i];
                        A[i] = u * c[i] - v * sn[i];
                        B[i] = u * sn[i] + v * c[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float u = A[2 * i], v = A[2 * i + 1], y = B[2 * i], z = B[2 * i + 1];
                        A[2 * i] = u * c[i] - v * sn[i];         A[2 * i + 1] = u * sn[i] + v * c[i];
                        B[2 * i] = y * c[2 + i] - z * sn[2 + i]; B[2 * i + 1] = y * sn[2 + i] + z * c[2 + i];
                    }
                }
            }
        }
        if (x.kind == 0) {
            float * o = (float *)(a.qo + x.t * a.qo_nb1 + x.r * a.qo_nb2 + x.i3 * a.qo_nb3);
            if (in) { *(v4f *)(o + ea) = v4f{A[0], A[1], A[2], A[3]}; *(v4f *)(o + eb) = v4f{B[0], B[1], B[2], B[3]}; }
            continue;
        }
        const int64_t row = a.rows ? *(const int32_t *)(a.rows + x.t * a.rows_nb1 + x.r * a.rows_nb2 + x.i3 * a.rows_nb3) : x.t;
        const bool stored = row >= 0 && row < a.n_rows;                   // as SET_ROWS: an index outside the cache stores nothing
        char * o = x.kind == 2 ? a.vo + row * a.vo_nb1 + x.r * a.vo_nb2 + x.i3 * a.vo_nb3 : a.ko + row * a.ko_nb1 + x.r * a.ko_nb2 + x.i3 * a.ko_nb3;
        const bool mine = (x.kind == 2 ? vin : in) && stored;
        const int pa = x.kind == 2 ? 8 * j : ea, pb = x.kind == 2 ? 8 * j + 4 : eb;
        if constexpr (!quant) {
            if (mine) { qn_store4<TYPE>(o, pa, A); qn_store4<TYPE>(o, pb, B); }
        } else {
            // a block is 32 consecutive values: through LDS, then a lane per block
            float * xs = cs + tt * 2 * half + g * 8 * L;
            *(v4f *)(xs + pa) = v4f{A[0], A[1], A[2], A[3]};
            *(v4f *)(xs + pb) = v4f{B[0], B[1], B[2], B[3]};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (stored && j < (x.kind == 2 ? a.dv : a.d) / 32) quant_block<TYPE>(xs + 32 * j, (uint8_t *)o + QBlk<TYPE>::bytes * j);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (x.kind == 1 && j == 0 && stored) {
            if (a.slot_pos)  ((int32_t *)(a.slot_pos + x.r * a.sp_nb2 + x.i3 * a.sp_nb3))[row] = *(const int32_t *)(a.pos + x.t * a.pos_nb1 + x.i3 * a.pos_nb3);
            if (a.slot_mass) ((float *)(a.slot_mass + x.r * a.sm_nb2 + x.i3 * a.sm_nb3))[row] = 0.0f;
        }
    }
}

template <int TYPE, int L> static int qn_launch_l(const QnArgs & a, hipStream_t s) {
    // 4 tokens a workgroup share its sines while that leaves 1024 workgroups; a few tokens are spread over as many workgroups as they have rows for
    const int64_t T = (int64_t)a.n * a.ne3, R = a.n_head + (a.vo ? 2 : 1) * a.n_head_kv, G = QN_THREADS / L;
    const int tt = T >= 4096 ? 4 : 1;
    const int64_t most = (tt * R + G - 1) / G, groups = (T + tt - 1) / tt;
    int64_t chunks = groups >= 1024 ? 1 : 1024 / groups;
    if (chunks > most) chunks = most;
    const size_t lds = ((size_t)tt * a.n_dims + (TYPE == MI355_TYPE_Q8_0 || TYPE == MI355_TYPE_Q4_0 ? QN_THREADS * 8 : 0)) * sizeof(float);
    MI355_LAUNCH("qk_norm_rope", (qk_norm_rope_kernel<TYPE, L>), dim3((unsigned)(groups * chunks)), dim3(QN_THREADS), lds, s, a, tt, (int)chunks);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
template <int TYPE> static int qn_launch(const QnArgs & a, hipStream_t s) {
    const int d = a.vo && a.dv > a.d ? a.dv : a.d;
    return d <= 64 ? qn_launch_l<TYPE, 8>(a, s) : d <= 128 ? qn_launch_l<TYPE, 16>(a, s) : qn_launch_l<TYPE, 32>(a, s);
}

} // namespace

extern "C" {

int mi355_qk_norm_rope(const mi355_qk_norm_rope_args * p, void * stream) {
    if (!p) return MI355_E_NULL;
    if (p->n != 0 && p->ne3 != 0) {                   // (tensors of no tokens or sequences, and caches of no rows, have no address)
        if (!p->q || !p->k || !p->q_out || !p->pos) return MI355_E_NULL;
        if (p->n_rows != 0 && (!p->k_out || !p->v != !p->v_out)) return MI355_E_NULL;
    }
    const int64_t dv = p->dv ? p->dv : p->head_dim;
    if (p->head_dim < 8 || p->head_dim > 256 || p->head_dim % 8 || dv < 8 || dv > 256 || dv % 8) return MI355_E_UNSUPPORTED;
    if (p->n_dims < 0 || p->n_dims > p->head_dim) return MI355_E_SHAPE;
    if (p->n_dims % 8 || (p->mode != 0 && p->mode != 2)) return MI355_E_UNSUPPORTED;
    const bool quant = p->type_kv == MI355_TYPE_Q8_0 || p->type_kv == MI355_TYPE_Q4_0;
    if (!quant && p->type_kv != MI355_TYPE_F32 && p->type_kv != MI355_TYPE_F16 && p->type_kv != MI355_TYPE_BF16) return MI355_E_TYPE;
    if (quant && (p->head_dim % 32 || (p->v && dv % 32))) return MI355_E_SHAPE;
    if (p->n < 0 || p->ne3 < 0 || p->n_head < 1 || p->n_head_kv < 1 || p->n_rows < 0) return MI355_E_SHAPE;
    if (p->n > (1 << 24) || p->ne3 > (1 << 24) || p->n * p->ne3 > (1 << 24) || p->n_head > 16384 || p->n_head_kv > 16384) return MI355_E_SHAPE;
    if (p->n_dims > 0 && (!(p->freq_base > 0.0f) || !(p->freq_scale > 0.0f) || (p->ext_factor != 0.0f && p->n_ctx_orig < 1))) return MI355_E_SHAPE;
    const int64_t f32s = (int64_t)(uintptr_t)p->q | p->q_nb1 | p->q_nb2 | p->q_nb3 | (int64_t)(uintptr_t)p->k | p->k_nb1 | p->k_nb2 | p->k_nb3 |
                         (int64_t)(uintptr_t)p->v | p->v_nb1 | p->v_nb2 | p->v_nb3 | (int64_t)(uintptr_t)p->q_out | p->qo_nb1 | p->qo_nb2 | p->qo_nb3 |
                         (int64_t)(uintptr_t)p->q_norm | (int64_t)(uintptr_t)p->k_norm;
    const int64_t cache = (int64_t)(uintptr_t)p->k_out | p->ko_nb1 | p->ko_nb2 | p->ko_nb3 | (int64_t)(uintptr_t)p->v_out | p->vo_nb1 | p->vo_nb2 | p->vo_nb3;
    const int64_t words = (int64_t)(uintptr_t)p->pos | p->pos_nb1 | p->pos_nb3 | (int64_t)(uintptr_t)p->rows | p->rows_nb1 | p->rows_nb2 | p->rows_nb3 |
                          (int64_t)(uintptr_t)p->freq_factors | (int64_t)(uintptr_t)p->slot_pos | p->sp_nb2 | p->sp_nb3 |
                          (int64_t)(uintptr_t)p->slot_mass | p->sm_nb2 | p->sm_nb3;
    if ((f32s & 15) || (cache & (quant ? 1 : 15)) || (words & 3)) return MI355_E_ALIGN;
    if (p->n == 0 || p->ne3 == 0) return MI355_OK;
    // q_out is q itself, row for row, or shares no memory with what is read: another order of q's rows would be written before they are read
    const Span qo(p->q_out, p->head_dim * 4, p->n, p->qo_nb1, p->n_head, p->qo_nb2, p->ne3, p->qo_nb3), q(p->q, p->head_dim * 4, p->n, p->q_nb1, p->n_head, p->q_nb2, p->ne3, p->q_nb3);
    if (!qo.same(q) && (spans_meet(qo, q) || spans_meet(qo, Span(p->k, p->head_dim * 4, p->n, p->k_nb1, p->n_head_kv, p->k_nb2, p->ne3, p->k_nb3)) ||
                        spans_meet(qo, Span(p->v, dv * 4, p->n, p->v_nb1, p->n_head_kv, p->v_nb2, p->ne3, p->v_nb3)))) return MI355_E_UNSUPPORTED;
    // and no place is written twice: heads, tokens and sequences of q_out lie apart, so do those of a cache whose rows are the tokens' own.  (Rows that
    // are given may share a pool: heads or sequences at one address, in rows of their own)
    const int64_t rk = mi355_row_size(p->type_kv, p->head_dim), rv = mi355_row_size(p->type_kv, dv), n1 = p->n < p->n_rows ? p->n : p->n_rows;
    if (qo.folds() || (!p->rows && Span(p->k_out, rk, n1, p->ko_nb1, p->n_head_kv, p->ko_nb2, p->ne3, p->ko_nb3).folds()) ||
        (!p->rows && p->v && Span(p->v_out, rv, n1, p->vo_nb1, p->n_head_kv, p->vo_nb2, p->ne3, p->vo_nb3).folds())) return MI355_E_UNSUPPORTED;

    QnArgs a;
    a.q = (const char *)p->q; a.q_nb1 = p->q_nb1; a.q_nb2 = p->q_nb2; a.q_nb3 = p->q_nb3;
    a.k = (const char *)p->k; a.k_nb1 = p->k_nb1; a.k_nb2 = p->k_nb2; a.k_nb3 = p->k_nb3;
    a.v = (const char *)p->v; a.v_nb1 = p->v_nb1; a.v_nb2 = p->v_nb2; a.v_nb3 = p->v_nb3;
    a.qw = p->q_norm; a.kw = p->k_norm; a.ff = p->freq_factors;
    a.qo = (char *)p->q_out; a.qo_nb1 = p->qo_nb1; a.qo_nb2 = p->qo_nb2; a.qo_nb3 = p->qo_nb3;
    a.ko = (char *)p->k_out; a.ko_nb1 = p->ko_nb1; a.ko_nb2 = p->ko_nb2; a.ko_nb3 = p->ko_nb3;
    a.vo = p->v ? (char *)p->v_out : nullptr; a.vo_nb1 = p->vo_nb1; a.vo_nb2 = p->vo_nb2; a.vo_nb3 = p->vo_nb3;
    a.pos = (const char *)p->pos; a.pos_nb1 = p->pos_nb1; a.pos_nb3 = p->pos_nb3;
    a.rows = (const char *)p->rows; a.rows_nb1 = p->rows_nb1; a.rows_nb2 = p->rows_nb2; a.rows_nb3 = p->rows_nb3;
    a.slot_pos = (char *)p->slot_pos; a.sp_nb2 = p->sp_nb2; a.sp_nb3 = p->sp_nb3;
    a.slot_mass = (char *)p->slot_mass; a.sm_nb2 = p->sm_nb2; a.sm_nb3 = p->sm_nb3;
    a.n_rows = p->n_rows;
    a.log2_step = p->n_dims > 0 ? 2.0 / p->n_dims * log2((double)p->freq_base) : 0.0;
    const RopeP rp = rope_params(p->n_dims > 0 ? p->n_dims : 8, p->mode, p->head_dim, p->n_ctx_orig > 0 ? p->n_ctx_orig : 1, p->freq_base, p->freq_scale,
                                 p->ext_factor, p->attn_factor, p->beta_fast, p->beta_slow);
    a.corr0 = rp.corr0; a.corr1 = rp.corr1;
    a.eps = p->eps; a.freq_scale = p->freq_scale; a.ext_factor = p->ext_factor;
    a.mscale = p->ext_factor != 0.0f ? p->attn_factor * (1.0f + 0.1f * logf(1.0f / p->freq_scale)) : p->attn_factor;
    a.d = (int)p->head_dim; a.dv = (int)dv; a.n_dims = p->n_dims; a.neox = p->mode == 2;
    a.n_head = (int)p->n_head; a.n_head_kv = (int)p->n_head_kv; a.n = (int)p->n; a.ne3 = (int)p->ne3;
    hipStream_t s = (hipStream_t)stream;
    switch (p->type_kv) {
        case MI355_TYPE_F32:  return qn_launch<MI355_TYPE_F32>(a, s);
        case MI355_TYPE_F16:  return qn_launch<MI355_TYPE_F16>(a, s);
        case MI355_TYPE_BF16: return qn_launch<MI355_TYPE_BF16>(a, s);
        case MI355_TYPE_Q8_0: return qn_launch<MI355_TYPE_Q8_0>(a, s);
    }
    return qn_launch<MI355_TYPE_Q4_0>(a, s);
}

} // extern "C"
