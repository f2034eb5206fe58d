// kv_evict.hip -- which slots of a bounded KV cache to keep, by the attention weight they have drawn (mi355_kv_evict).
//
// Per (sequence, KV head): the n_keep slots with the largest key, ties to the lower slot; key = the slot's mass, or +inf where its position
// is one of the first n_sink or the newest n_recent (NaN counts as -inf, -0 as +0).  A radix search over the 32-bit images of the keys
// (order-preserving: sign flipped for positive floats, all bits for negative ones) finds the n_keep-th largest and how many of its equals
// belong to the kept ones; one ordered pass then writes both index lists ascending.  All integer work: the result does not depend on
// timing.  The rows are gathered by a second launch.
#include "common.h"

namespace {

struct KeArgs {
    const char * mass, * pos, * n_used, * n_past;
    int64_t mass_nb2, mass_nb3, pos_nb2, pos_nb3;
    char * kept, * evicted;
    int64_t kept_nb2, kept_nb3, ev_nb2, ev_nb3;
    char * mass_out, * pos_out;
    int64_t mo_nb2, mo_nb3, po_nb2, po_nb3;
    int n_kv, n_keep, n_evict, n_sink, n_recent, n_head_kv;
};

constexpr int KE_THREADS = 1024, KE_WAVES = KE_THREADS / 64;

static __device__ __forceinline__ uint32_t ke_key(float m, bool keep) {
    if (keep) return 0xff800000u;                     // the image of +inf
    if (m != m) m = -INFINITY;
    if (m == 0.0f) m = 0.0f;                          // -0 and +0 are equal
    const uint32_t u = __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive prefix sum of a flag over the workgroup; `total` for every thread
static __device__ __forceinline__ int ke_prefix(bool f, int * sh, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t b = __ballot(f);
    __syncthreads();
    if (lane == 0) sh[wave] = __popcll(b);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < KE_WAVES; w++) { before += w < wave ? sh[w] : 0; all += sh[w]; }
    total = all;
    return before + __popcll(b & ((1ull << lane) - 1));
}

__global__ void __launch_bounds__(KE_THREADS)
kv_select_kernel(const KeArgs a) {
    __shared__ int hist[256], sh[KE_WAVES], pick[2];
    const int tid = threadIdx.x, hk = blockIdx.x, i3 = blockIdx.y;
    const float * mass = (const float *)(a.mass + hk * a.mass_nb2 + i3 * a.mass_nb3);
    const int32_t * pos = (const int32_t *)(a.pos + hk * a.pos_nb2 + i3 * a.pos_nb3);
    int32_t * kept = (int32_t *)(a.kept + hk * a.kept_nb2 + i3 * a.kept_nb3);
    int32_t * evicted = a.evicted ? (int32_t *)(a.evicted + hk * a.ev_nb2 + i3 * a.ev_nb3) : nullptr;
    int n = a.n_used ? ((const int32_t *)a.n_used)[i3] : a.n_kv;
    n = n < 0 ? 0 : n < a.n_kv ? n : a.n_kv;
    const int64_t recent = (int64_t)((const int32_t *)a.n_past)[i3] - a.n_recent;
    auto key = [&](int j) { const int p = pos[j]; return ke_key(mass[j], p < a.n_sink || p >= recent); };

    // the smallest kept key T and the number of kept slots that equal it
    uint32_t T = 0;
    int equal = 0x7fffffff;
    if (n > a.n_keep) {
        int want = a.n_keep;                          // rank of the wanted key, counted from the largest
        uint32_t mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += KE_THREADS) { const uint32_t k = key(j); if ((k & mask) == T) atomicAdd(&hist[k >> shift & 255], 1); }
            __syncthreads();
            if (tid == 0) {
                int c = 0, b = 255;
                while (b > 0 && c + hist[b] < want) { c += hist[b]; b--; }
                pick[0] = b; pick[1] = want - c;
            }
            __syncthreads();
            T |= (uint32_t)pick[0] << shift;
            want = pick[1];
            mask |= 255u << shift;
            __syncthreads();
        }
        equal = want;
    }
    // one ordered pass: slot j stays if its key is above T, or equals T and fewer than `equal` equals lie before it
    int kept_n = 0, eq_n = 0, ev_n = 0;
    for (int j0 = 0; j0 < n; j0 += KE_THREADS) {
        const int j = j0 + tid;
        const uint32_t k = j < n ? key(j) : 0;
        int t_eq, t_keep, t_ev;
        const bool eq = j < n && k == T;
        const int p_eq = ke_prefix(eq, sh, t_eq);
        const bool keep = j < n && (k > T || (eq && eq_n + p_eq < equal));
        const int p_keep = ke_prefix(keep, sh, t_keep);
        const bool ev = j < n && !keep;
        const int p_ev = ke_prefix(ev, sh, t_ev);
        if (keep) kept[kept_n + p_keep] = j;
        if (ev && evicted && ev_n + p_ev < a.n_evict) evicted[ev_n + p_ev] = j;
        eq_n += t_eq; kept_n += t_keep; ev_n += t_ev;
    }
    for (int j = kept_n + tid; j < a.n_keep; j += KE_THREADS) kept[j] = -1;
    if (evicted) for (int j = ev_n + tid; j < a.n_evict; j += KE_THREADS) evicted[j] = -1;
}

struct KgArgs {
    const char * kept;
    int64_t kept_nb2, kept_nb3;
    const char * src[2]; char * dst[2];
    int64_t s_nb1[2], s_nb2[2], s_nb3[2], d_nb1[2], d_nb2[2], d_nb3[2];
    int row_bytes[2], n_keep, n_head_kv;
    const char * mass, * pos;
    int64_t mass_nb2, mass_nb3, pos_nb2, pos_nb3;
    char * mass_out, * pos_out;
    int64_t mo_nb2, mo_nb3, po_nb2, po_nb3;
};

// one wave per kept slot: the K and V rows in 2-byte pieces, the tables' entries
__global__ void __launch_bounds__(256)
kv_gather_kernel(const KgArgs a) {
    const int lane = threadIdx.x & 63, hk = blockIdx.y, i3 = blockIdx.z;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.n_keep) return;
    const int j = ((const int32_t *)(a.kept + hk * a.kept_nb2 + i3 * a.kept_nb3))[i];
    if (lane == 0) {
        if (a.mass_out) ((float *)(a.mass_out + hk * a.mo_nb2 + i3 * a.mo_nb3))[i] = j < 0 ? 0.0f : ((const float *)(a.mass + hk * a.mass_nb2 + i3 * a.mass_nb3))[j];
        if (a.pos_out) ((int32_t *)(a.pos_out + hk * a.po_nb2 + i3 * a.po_nb3))[i] = j < 0 ? -1 : ((const int32_t *)(a.pos + hk * a.pos_nb2 + i3 * a.pos_nb3))[j];
    }
    if (j < 0) return;
    for (int s = 0; s < 2; s++) {
        if (!a.src[s]) continue;
        const uint16_t * x = (const uint16_t *)(a.src[s] + j * a.s_nb1[s] + hk * a.s_nb2[s] + i3 * a.s_nb3[s]);
        uint16_t * y = (uint16_t *)(a.dst[s] + i * a.d_nb1[s] + hk * a.d_nb2[s] + i3 * a.d_nb3[s]);
        for (int e = lane; e < a.row_bytes[s] / 2; e += 64) y[e] = x[e];
    }
}

} // namespace

extern "C" {

int mi355_kv_evict(const mi355_kv_evict_args * p, void * stream) {
    if (!p || (p->n_kv > 0 && (!p->mass || !p->slot_pos)) || !p->n_past || !p->kept) return MI355_E_NULL;
    if (!p->k != !p->k_out || !p->v != !p->v_out) return MI355_E_NULL;
    if (p->n_kv < 0 || p->n_kv > 0x7fffffff || p->n_keep < 1 || p->n_keep > 0x7fffffff || p->n_evict < 0 || p->n_evict > 0x7fffffff) return MI355_E_SHAPE;
    if (p->n_sink < 0 || p->n_recent < 0 || (int64_t)p->n_sink + p->n_recent > p->n_keep) return MI355_E_SHAPE;
    if (p->n_head_kv < 1 || p->n_head_kv > 65535 || p->ne3 < 0 || p->ne3 > 65535) return MI355_E_SHAPE;
    const int64_t dv = p->dv ? p->dv : p->d;
    if (p->k || p->v) {
        if (mi355_blck_size(p->type_kv) == 0) return MI355_E_TYPE;
        if (p->type_kv != MI355_TYPE_F32 && p->type_kv != MI355_TYPE_F16 && p->type_kv != MI355_TYPE_BF16 && p->type_kv != MI355_TYPE_Q8_0 && p->type_kv != MI355_TYPE_Q4_0) return MI355_E_TYPE;
        if (p->d < 1 || p->d > (1 << 20) || dv < 1 || dv > (1 << 20) || mi355_row_size(p->type_kv, p->d) < 0 || mi355_row_size(p->type_kv, dv) < 0) return MI355_E_SHAPE;
    }
    const int64_t words = (int64_t)(uintptr_t)p->mass | p->mass_nb2 | p->mass_nb3 | (int64_t)(uintptr_t)p->slot_pos | p->pos_nb2 | p->pos_nb3 |
                          (int64_t)(uintptr_t)p->n_used | (int64_t)(uintptr_t)p->n_past | (int64_t)(uintptr_t)p->kept | p->kept_nb2 | p->kept_nb3 |
                          (int64_t)(uintptr_t)p->evicted | p->ev_nb2 | p->ev_nb3 | (int64_t)(uintptr_t)p->mass_out | p->mo_nb2 | p->mo_nb3 |
                          (int64_t)(uintptr_t)p->pos_out | p->po_nb2 | p->po_nb3;
    const int64_t rows = (int64_t)(uintptr_t)p->k | p->k_nb1 | p->k_nb2 | p->k_nb3 | (int64_t)(uintptr_t)p->v | p->v_nb1 | p->v_nb2 | p->v_nb3 |
                         (int64_t)(uintptr_t)p->k_out | p->ko_nb1 | p->ko_nb2 | p->ko_nb3 | (int64_t)(uintptr_t)p->v_out | p->vo_nb1 | p->vo_nb2 | p->vo_nb3;
    if ((words & 3) || ((p->k || p->v) && (rows & 1))) return MI355_E_ALIGN;
    // the gathered rows and tables go to other memory: a slot may be read after its place has been written
    if ((p->k && p->k == p->k_out) || (p->v && p->v == p->v_out) || (p->mass_out && p->mass_out == p->mass) || (p->pos_out && p->pos_out == p->slot_pos)) return MI355_E_UNSUPPORTED;
    if (p->ne3 == 0) return MI355_OK;

    KeArgs a;
    a.mass = (const char *)p->mass; a.mass_nb2 = p->mass_nb2; a.mass_nb3 = p->mass_nb3;
    a.pos = (const char *)p->slot_pos; a.pos_nb2 = p->pos_nb2; a.pos_nb3 = p->pos_nb3;
    a.n_used = (const char *)p->n_used; a.n_past = (const char *)p->n_past;
    a.kept = (char *)p->kept; a.kept_nb2 = p->kept_nb2; a.kept_nb3 = p->kept_nb3;
    a.evicted = (char *)p->evicted; a.ev_nb2 = p->ev_nb2; a.ev_nb3 = p->ev_nb3;
    a.n_kv = (int)p->n_kv; a.n_keep = (int)p->n_keep; a.n_evict = (int)p->n_evict; a.n_sink = p->n_sink; a.n_recent = p->n_recent; a.n_head_kv = (int)p->n_head_kv;
    hipStream_t s = (hipStream_t)stream;
    MI355_LAUNCH("kv_select", kv_select_kernel, dim3((unsigned)p->n_head_kv, (unsigned)p->ne3), dim3(KE_THREADS), 0, s, a);
    MI355_CHECK_LAUNCH();
    if (!p->k && !p->v && !p->mass_out && !p->pos_out) return MI355_OK;

    KgArgs g;
    g.kept = a.kept; g.kept_nb2 = a.kept_nb2; g.kept_nb3 = a.kept_nb3;
    g.src[0] = (const char *)p->k; g.s_nb1[0] = p->k_nb1; g.s_nb2[0] = p->k_nb2; g.s_nb3[0] = p->k_nb3;
    g.dst[0] = (char *)p->k_out; g.d_nb1[0] = p->ko_nb1; g.d_nb2[0] = p->ko_nb2; g.d_nb3[0] = p->ko_nb3;
    g.src[1] = (const char *)p->v; g.s_nb1[1] = p->v_nb1; g.s_nb2[1] = p->v_nb2; g.s_nb3[1] = p->v_nb3;
    g.dst[1] = (char *)p->v_out; g.d_nb1[1] = p->vo_nb1; g.d_nb2[1] = p->vo_nb2; g.d_nb3[1] = p->vo_nb3;
    g.row_bytes[0] = p->k ? (int)mi355_row_size(p->type_kv, p->d) : 0; g.row_bytes[1] = p->v ? (int)mi355_row_size(p->type_kv, dv) : 0;
    g.n_keep = a.n_keep; g.n_head_kv = a.n_head_kv;
    g.mass = a.mass; g.mass_nb2 = a.mass_nb2; g.mass_nb3 = a.mass_nb3; g.pos = a.pos; g.pos_nb2 = a.pos_nb2; g.pos_nb3 = a.pos_nb3;
    g.mass_out = (char *)p->mass_out; g.mo_nb2 = p->mo_nb2; g.mo_nb3 = p->mo_nb3;
    g.pos_out = (char *)p->pos_out; g.po_nb2 = p->po_nb2; g.po_nb3 = p->po_nb3;
    MI355_LAUNCH("kv_gather", kv_gather_kernel, dim3((unsigned)((a.n_keep + 3) / 4), (unsigned)p->n_head_kv, (unsigned)p->ne3), dim3(256), 0, s, g);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}

} // extern "C"
