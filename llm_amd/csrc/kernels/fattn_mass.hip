// fattn_mass.hip -- attention weight per cached slot: mi355_flash_attn_ext_mass (a decode step's attention together with it) and
// mi355_attn_mass (the weight alone, for any number of queries).
//
//   s_ij = scale q_i . k_j [softcap] + slope mask_ij      p_ij = exp(s_ij - m_i) / l_i     (m_i, l_i: maximum and sum over the slots i sees)
//   dst_i = sum_j p_ij v_j      mass_out[hk][j] = decay mass_in[hk][j] + sum over the heads of hk and all queries i of p_ij
// A slot that a query does not see (mask -inf) takes no part whatever its row holds, NaN included; a query that sees nothing gives a zero row and
// no weight.  Everything between the cache's own values and the f32 results is f32.
#include "common.h"

namespace {

struct MArgs {
    const char * q; int64_t q_nb1, q_nb2, q_nb3;
    const char * k; int64_t k_nb1, k_nb2, k_nb3;
    const char * v; int64_t v_nb1, v_nb2, v_nb3;
    const char * mask; int64_t m_nb1, m_nb2, m_nb3, m_ne2, m_ne3;
    char * dst; int64_t d_nb1, d_nb2, d_nb3;
    const char * mass_in; int64_t in_nb2, in_nb3;
    char * mass_out; int64_t out_nb2, out_nb3;
    int n_q, n_kv, n_head, n_head_kv, d, dv;
    float scale, max_bias, logit_softcap, m0, m1, decay;
    uint32_t n_head_log2;
    float * logits;     // [ne3][n_head][n_q][n_kv] (with dst), else NULL
    float * stats;      // [ne3][n_head][n_q][2]: m, 1 / l (0: sees nothing)
};

constexpr int MT = 256;

template <int TYPE> static __device__ __forceinline__ float kv_value(const char * row, int e) {
    if (TYPE == MI355_TYPE_F16) return h2f(((const uint16_t *)row)[e]);
    if (TYPE == MI355_TYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t *)row)[e] << 16);
    if (TYPE == MI355_TYPE_Q8_0) { const char * b = row + (e >> 5) * 34; return h2f(*(const uint16_t *)b) * (float)((const int8_t *)(b + 2))[e & 31]; }
    const char * b = row + (e >> 5) * 18;
    const int n = ((const uint8_t *)(b + 2))[e & 15] >> ((e & 16) ? 4 : 0) & 15;
    return h2f(*(const uint16_t *)b) * (float)(n - 8);
}

static __device__ __forceinline__ float m_slope(const MArgs & a, uint32_t h) {
    if (!(a.max_bias > 0.0f)) return 1.0f;
    return h < a.n_head_log2 ? powf(a.m0, h + 1) : powf(a.m1, 2 * (h - a.n_head_log2) + 1);
}

// logit of slot j for a query row in LDS; -inf where the mask hides the slot
template <int TYPE> static __device__ __forceinline__ float logit(const MArgs & a, const float * q, const char * krow, const char * mrow, float slope, int j) {
    const float mv = mrow ? slope * h2f(((const uint16_t *)mrow)[j]) : 0.0f;
    if (mv == -INFINITY) return -INFINITY;
    float t = 0.0f;
    for (int e = 0; e < a.d; e++) t = __builtin_fmaf(q[e], kv_value<TYPE>(krow, e), t);
    t = a.logit_softcap != 0.0f ? a.logit_softcap * tanhf(t * (a.scale / a.logit_softcap)) : t * a.scale;
    return t + mv;
}

// one workgroup per (query, head, sequence): statistics, and with dst the attention row
template <int TYPE>
__global__ void __launch_bounds__(MT)
mass_rows_kernel(const MArgs a) {
    __shared__ float q[256], sh[MT / 64], shm[MT / 64];
    const int tid = threadIdx.x, h = blockIdx.x, iq = blockIdx.y, i3 = blockIdx.z;
    const int hk = h / (a.n_head / a.n_head_kv);
    const float * qr = (const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3);
    if (tid < a.d) q[tid] = qr[tid];
    __syncthreads();
    const char * kb = a.k + hk * a.k_nb2 + i3 * a.k_nb3;
    const char * mrow = a.mask ? a.mask + iq * a.m_nb1 + (h % a.m_ne2) * a.m_nb2 + (i3 % a.m_ne3) * a.m_nb3 : nullptr;
    const float slope = m_slope(a, h);
    const int64_t row = ((int64_t)i3 * a.n_head + h) * a.n_q + iq;
    float * lg = a.logits ? a.logits + row * a.n_kv : nullptr;
    float m = -INFINITY, l = 0.0f;
    for (int j = tid; j < a.n_kv; j += MT) {
        const float s = logit<TYPE>(a, q, kb + (int64_t)j * a.k_nb1, mrow, slope, j);
        if (lg) lg[j] = s;
        if (s == -INFINITY) continue;
        const float mn = fmaxf(m, s);
        l = l * expf(m - mn) + expf(s - mn);
        m = mn;
    }
    float M = m;
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((tid & 63) == 0) shm[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(shm[0], shm[1]), fmaxf(shm[2], shm[3]));
    const float L = block_sum_n<MT / 64>(m == -INFINITY ? l : l * expf(m - M), sh);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (tid == 0) { a.stats[row * 2] = M; a.stats[row * 2 + 1] = inv; }
    if (!a.dst) return;
    __syncthreads();
    float * o = (float *)(a.dst + h * a.d_nb1 + iq * a.d_nb2 + i3 * a.d_nb3);
    const char * vb = a.v + hk * a.v_nb2 + i3 * a.v_nb3;
    for (int e = tid; e < a.dv; e += MT) {
        float t = 0.0f;
        for (int j = 0; j < a.n_kv; j++) {
            const float s = lg[j];
            if (s != -INFINITY) t = __builtin_fmaf(expf(s - M), kv_value<TYPE>(vb + (int64_t)j * a.v_nb1, e), t);
        }
        o[e] = t * inv;
    }
}

// one thread per slot: its weight over the heads and queries of its KV head
template <int TYPE>
__global__ void __launch_bounds__(MT)
mass_slots_kernel(const MArgs a) {
    __shared__ float q[256];
    const int tid = threadIdx.x, j = blockIdx.x * MT + tid, hk = blockIdx.y, i3 = blockIdx.z;
    const int ratio = a.n_head / a.n_head_kv;
    const char * krow = a.k + (int64_t)(j < a.n_kv ? j : 0) * a.k_nb1 + hk * a.k_nb2 + i3 * a.k_nb3;
    float t = 0.0f;
    for (int h = hk * ratio; h < hk * ratio + ratio; h++)
        for (int iq = 0; iq < a.n_q; iq++) {
            const int64_t row = ((int64_t)i3 * a.n_head + h) * a.n_q + iq;
            float s = -INFINITY;
            if (a.logits) {
                if (j < a.n_kv) s = a.logits[row * a.n_kv + j];
            } else {
                __syncthreads();
                if (tid < a.d) q[tid] = ((const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3))[tid];
                __syncthreads();
                const char * mrow = a.mask ? a.mask + iq * a.m_nb1 + (h % a.m_ne2) * a.m_nb2 + (i3 % a.m_ne3) * a.m_nb3 : nullptr;
                if (j < a.n_kv) s = logit<TYPE>(a, q, krow, mrow, m_slope(a, h), j);
            }
            if (s != -INFINITY) t += expf(s - a.stats[row * 2]) * a.stats[row * 2 + 1];
        }
    if (j >= a.n_kv) return;
    if (a.mass_in) t += a.decay * ((const float *)(a.mass_in + hk * a.in_nb2 + i3 * a.in_nb3))[j];
    ((float *)(a.mass_out + hk * a.out_nb2 + i3 * a.out_nb3))[j] = t;
}

template <int TYPE> static int mass_launch(const MArgs & a, int ne3, hipStream_t s) {
    MI355_LAUNCH("fattn_mass_rows", mass_rows_kernel<TYPE>, dim3((unsigned)a.n_head, (unsigned)a.n_q, (unsigned)ne3), dim3(MT), 0, s, a);
    MI355_CHECK_LAUNCH();
    if (a.n_kv == 0) return MI355_OK;
    MI355_LAUNCH("fattn_mass", mass_slots_kernel<TYPE>, dim3((unsigned)((a.n_kv + MT - 1) / MT), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(MT), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}

static int64_t mass_workspace(const mi355_fattn_args * p, bool with_dst) {
    if (!p || p->n_q < 0 || p->n_kv < 0 || p->n_head < 0 || p->ne3 < 0) return -1;
    const int64_t rows = p->ne3 * p->n_head * p->n_q;
    return rows * 8 + (with_dst ? rows * p->n_kv * 4 : 0);
}

static int mass_run(const mi355_fattn_args * p, const mi355_attn_mass_args * w, bool with_dst, void * workspace, int64_t workspace_bytes, void * stream) {
    if (!p || !w || !p->q || (p->n_kv > 0 && (!p->k || !w->mass_out)) || (with_dst && (!p->dst || (p->n_kv > 0 && !p->v)))) return MI355_E_NULL;
    const int64_t dv = p->dv ? p->dv : p->d;
    if (p->d < 8 || p->d > 256 || p->d % 8 != 0) return MI355_E_UNSUPPORTED;
    if (with_dst && (dv < 8 || dv > p->d || dv % 8 != 0)) return MI355_E_UNSUPPORTED;
    if (p->type_k != MI355_TYPE_F16 && p->type_k != MI355_TYPE_BF16 && p->type_k != MI355_TYPE_Q8_0 && p->type_k != MI355_TYPE_Q4_0) return MI355_E_TYPE;
    if (with_dst && p->type_v != p->type_k) return MI355_E_TYPE;
    const bool quant = p->type_k == MI355_TYPE_Q8_0 || p->type_k == MI355_TYPE_Q4_0;
    if (quant && (p->d % 32 != 0 || (with_dst && dv % 32 != 0))) return MI355_E_SHAPE;
    if (p->n_head < 1 || p->n_head > 65535 || p->n_head_kv < 1 || p->n_head % p->n_head_kv != 0 || p->n_q < 1 || p->n_q > 65535 || p->n_kv < 0 ||
        p->n_kv > (1 << 30) || p->ne3 < 1 || p->ne3 > 65535) return MI355_E_SHAPE;
    if (with_dst && p->n_q > MI355_MASS_MAX_Q) return MI355_E_UNSUPPORTED;
    if (p->mask && (p->m_ne2 < 1 || p->m_ne3 < 1)) return MI355_E_SHAPE;
    const int64_t f32s = (int64_t)(uintptr_t)p->q | p->q_nb1 | p->q_nb2 | p->q_nb3 |
                         (with_dst ? (int64_t)(uintptr_t)p->dst | p->d_nb1 | p->d_nb2 | p->d_nb3 : 0) | (int64_t)(uintptr_t)workspace;
    int64_t cache = (int64_t)(uintptr_t)p->k | p->k_nb1 | p->k_nb2 | p->k_nb3;
    if (with_dst) cache |= (int64_t)(uintptr_t)p->v | p->v_nb1 | p->v_nb2 | p->v_nb3;
    const int64_t words = (int64_t)(uintptr_t)w->mass_in | w->in_nb2 | w->in_nb3 | (int64_t)(uintptr_t)w->mass_out | w->out_nb2 | w->out_nb3;
    const int64_t halves = p->mask ? (int64_t)(uintptr_t)p->mask | p->m_nb1 | p->m_nb2 | p->m_nb3 : 0;
    if ((f32s & 15) || (cache & (quant ? 1 : 15)) || (words & 3) || (halves & 1)) return MI355_E_ALIGN;
    const int64_t need = mass_workspace(p, with_dst);
    if (need > 0 && (!workspace || workspace_bytes < need)) return MI355_E_WORKSPACE;

    MArgs a;
    a.q = (const char *)p->q; a.q_nb1 = p->q_nb1; a.q_nb2 = p->q_nb2; a.q_nb3 = p->q_nb3;
    a.k = (const char *)p->k; a.k_nb1 = p->k_nb1; a.k_nb2 = p->k_nb2; a.k_nb3 = p->k_nb3;
    a.v = (const char *)p->v; a.v_nb1 = p->v_nb1; a.v_nb2 = p->v_nb2; a.v_nb3 = p->v_nb3;
    a.mask = (const char *)p->mask; a.m_nb1 = p->m_nb1; a.m_nb2 = p->m_nb2; a.m_nb3 = p->m_nb3; a.m_ne2 = p->m_ne2; a.m_ne3 = p->m_ne3;
    a.dst = with_dst ? (char *)p->dst : nullptr; a.d_nb1 = p->d_nb1; a.d_nb2 = p->d_nb2; a.d_nb3 = p->d_nb3;
    a.mass_in = w->decay != 0.0f ? (const char *)w->mass_in : nullptr; a.in_nb2 = w->in_nb2; a.in_nb3 = w->in_nb3;
    a.mass_out = (char *)w->mass_out; a.out_nb2 = w->out_nb2; a.out_nb3 = w->out_nb3;
    a.n_q = (int)p->n_q; a.n_kv = (int)p->n_kv; a.n_head = (int)p->n_head; a.n_head_kv = (int)p->n_head_kv; a.d = (int)p->d; a.dv = (int)dv;
    a.scale = p->scale; a.max_bias = p->max_bias; a.logit_softcap = p->logit_softcap; a.decay = w->decay;
    a.n_head_log2 = 1u << (uint32_t)floorf(log2f((float)p->n_head));
    a.m0 = powf(2.0f, -(p->max_bias) / a.n_head_log2);
    a.m1 = powf(2.0f, -(p->max_bias / 2.0f) / a.n_head_log2);
    a.stats = (float *)workspace;
    a.logits = with_dst ? a.stats + p->ne3 * p->n_head * p->n_q * 2 : nullptr;
    hipStream_t s = (hipStream_t)stream;
    switch (p->type_k) {
        case MI355_TYPE_F16:  return mass_launch<MI355_TYPE_F16>(a, (int)p->ne3, s);
        case MI355_TYPE_BF16: return mass_launch<MI355_TYPE_BF16>(a, (int)p->ne3, s);
        case MI355_TYPE_Q8_0: return mass_launch<MI355_TYPE_Q8_0>(a, (int)p->ne3, s);
    }
    return mass_launch<MI355_TYPE_Q4_0>(a, (int)p->ne3, s);
}

} // namespace

extern "C" {

int64_t mi355_flash_attn_ext_mass_workspace_bytes(const mi355_fattn_args * p) { return mass_workspace(p, true); }

int mi355_flash_attn_ext_mass(const mi355_fattn_args * p, const mi355_attn_mass_args * w, void * workspace, int64_t workspace_bytes, void * stream) {
    return mass_run(p, w, true, workspace, workspace_bytes, stream);
}

int64_t mi355_attn_mass_workspace_bytes(const mi355_fattn_args * p) { return mass_workspace(p, false); }

int mi355_attn_mass(const mi355_fattn_args * p, const mi355_attn_mass_args * w, void * workspace, int64_t workspace_bytes, void * stream) {
    return mass_run(p, w, false, workspace, workspace_bytes, stream);
}

} // extern "C"
