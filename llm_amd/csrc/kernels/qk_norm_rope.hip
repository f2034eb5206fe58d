// qk_norm_rope.hip -- attention input of models that normalise queries and keys per head: RMS norm x weight and the position rotation of
// every q and k head, and the store of k and v into their cache rows, in one launch (mi355_qk_norm_rope).
//
//   y = x / sqrt(mean(x^2) + eps) * w            over a head's head_dim values
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = pos * f_i,  pairs (2i, 2i + 1) NORMAL, (i, i + n_dims / 2) NEOX
// Angles are formed and reduced to one turn in 64 bits: in 32 bits the product alone is off by 0.01 rad at position 10^5.
#include "row_formats.h"
#include "rope.h"

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

template <int TYPE> static __device__ __forceinline__ void qn_store(char * row, int e, float v) {
    if (TYPE == MI355_TYPE_F32)       ((float *)row)[e] = v;
    else if (TYPE == MI355_TYPE_F16)  ((__half *)row)[e] = cvt<float, __half>(v);
    else if (TYPE == MI355_TYPE_BF16) ((bf16_bits *)row)[e] = cvt<float, bf16_bits>(v);
}

// one wave per row (a head of q, k or v of one token)
template <int TYPE>
__global__ void __launch_bounds__(64)
qk_norm_rope_kernel(const QnArgs a) {
    __shared__ float x[256];
    const int lane = threadIdx.x;
    const int r = blockIdx.y, t = blockIdx.x % a.n, i3 = blockIdx.x / a.n;
    const bool is_q = r < a.n_head, is_v = r >= a.n_head + a.n_head_kv;
    const int hk = is_q ? 0 : is_v ? r - a.n_head - a.n_head_kv : r - a.n_head;
    const int d = is_v ? a.dv : a.d;
    const float * src = (const float *)(is_q ? a.q + t * a.q_nb1 + r * a.q_nb2 + i3 * a.q_nb3 : is_v ? a.v + t * a.v_nb1 + hk * a.v_nb2 + i3 * a.v_nb3
                                                                                                    : a.k + t * a.k_nb1 + hk * a.k_nb2 + i3 * a.k_nb3);
    const int pos = *(const int32_t *)(a.pos + t * a.pos_nb1 + i3 * a.pos_nb3);
    float ss = 0.0f;
    for (int e = lane; e < d; e += 64) { const float f = src[e]; x[e] = f; ss += f * f; }
    if (!is_v) {
        const float s = 1.0f / sqrtf(wave_sum(ss) / d + a.eps);
        const float * w = is_q ? a.qw : a.kw;
        for (int e = lane; e < d; e += 64) x[e] = x[e] * s * (w ? w[e] : 1.0f);
        __syncthreads();
        for (int i = lane; i < a.n_dims / 2; i += 64) {
            const int ia = a.neox ? i : 2 * i, ib = a.neox ? i + a.n_dims / 2 : 2 * i + 1;
            const double rev = (double)pos * qn_freq(a, i);
            float c, sn;
            sincospif(2.0f * (float)(rev - rint(rev)), &sn, &c);
            c *= a.mscale; sn *= a.mscale;
            const float xa = x[ia], xb = x[ib];
            x[ia] = xa * c - xb * sn;
            x[ib] = xa * sn + xb * c;
        }
    }
    __syncthreads();
    if (is_q) {
        float * o = (float *)(a.qo + t * a.qo_nb1 + r * a.qo_nb2 + i3 * a.qo_nb3);
        for (int e = lane; e < d; e += 64) o[e] = x[e];
        return;
    }
    const int64_t row = a.rows ? *(const int32_t *)(a.rows + t * a.rows_nb1 + hk * a.rows_nb2 + i3 * a.rows_nb3) : t;
    if (row < 0 || row >= a.n_rows) return;           // as SET_ROWS: an index outside the cache stores nothing
    char * o = is_v ? a.vo + row * a.vo_nb1 + hk * a.vo_nb2 + i3 * a.vo_nb3 : a.ko + row * a.ko_nb1 + hk * a.ko_nb2 + i3 * a.ko_nb3;
    if constexpr (TYPE == MI355_TYPE_Q8_0 || TYPE == MI355_TYPE_Q4_0) {
        if (lane < d / 32) quant_block<TYPE>(x + 32 * lane, (uint8_t *)o + QBlk<TYPE>::bytes * lane);
    } else {
        for (int e = lane; e < d; e += 64) qn_store<TYPE>(o, e, x[e]);
    }
    if (!is_v && lane == 0) {
        if (a.slot_pos)  ((int32_t *)(a.slot_pos + hk * a.sp_nb2 + i3 * a.sp_nb3))[row] = pos;
        if (a.slot_mass) ((float *)(a.slot_mass + hk * a.sm_nb2 + i3 * a.sm_nb3))[row] = 0.0f;
    }
}

template <int TYPE> static int qn_launch(const QnArgs & a, hipStream_t s) {
    const int rows = a.n_head + (a.vo ? 2 : 1) * a.n_head_kv;
    MI355_LAUNCH("qk_norm_rope", qk_norm_rope_kernel<TYPE>, dim3((unsigned)(a.n * a.ne3), (unsigned)rows), dim3(64), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}

} // namespace

extern "C" {

int mi355_qk_norm_rope(const mi355_qk_norm_rope_args * p, void * stream) {
    if (!p || !p->q || !p->k || !p->q_out || !p->k_out || !p->pos || !p->v != !p->v_out) return MI355_E_NULL;
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

    QnArgs a;
    a.q = (const char *)p->q; a.q_nb1 = p->q_nb1; a.q_nb2 = p->q_nb2; a.q_nb3 = p->q_nb3;
    a.k = (const char *)p->k; a.k_nb1 = p->k_nb1; a.k_nb2 = p->k_nb2; a.k_nb3 = p->k_nb3;
    a.v = (const char *)p->v; a.v_nb1 = p->v_nb1; a.v_nb2 = p->v_nb2; a.v_nb3 = p->v_nb3;
    a.qw = p->q_norm; a.kw = p->k_norm; a.ff = p->freq_factors;
    a.qo = (char *)p->q_out; a.qo_nb1 = p->qo_nb1; a.qo_nb2 = p->qo_nb2; a.qo_nb3 = p->qo_nb3;
    a.ko = (char *)p->k_out; a.ko_nb1 = p->ko_nb1; a.ko_nb2 = p->ko_nb2; a.ko_nb3 = p->ko_nb3;
    a.vo = (char *)p->v_out; a.vo_nb1 = p->vo_nb1; a.vo_nb2 = p->vo_nb2; a.vo_nb3 = p->vo_nb3;
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
