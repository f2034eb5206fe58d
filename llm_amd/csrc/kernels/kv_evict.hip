// kv_evict.hip -- which slots of a bounded KV cache to keep, by the attention weight they have drawn (mi355_kv_evict).
//
// Per (sequence, KV head): the n_keep slots with the largest key, ties to the lower slot; key = the slot's mass, or more than any mass where its
// position is one of the first n_sink or the newest n_recent, pinned (NaN counts as -inf, -0 as +0).  The keys' 32-bit images (order-preserving: sign
// flipped for positive floats, all bits for negative ones) are searched for the n_keep-th largest; one ordered pass then writes both index
// lists ascending.  All integer work: the result does not depend on timing.  The rows are gathered by a second launch.
//
// Bound by latency: one workgroup per head has to agree on every step of the search.  A step parts the range of keys that can still hold the
// wanted one into 2048 buckets (an LDS histogram), so three steps settle 32 bits, and masses, which spread over the range as logarithms do,
// seldom meet in a bucket; the pinned slots are counted aside, and a wave whose lanes all fall into one bucket adds once.
// Up to 32768 slots the keys stay in registers; beyond, every step reads them again.  2049 slots x 128 heads 10.9 us, 32768 x 8
// heads 31 us (8 of them loading 256 KB on each of 8 CUs, 7 writing the lists) and 10.6 us for the rows.
// (Digits of 8 bits from the top, keys re-read: 54 / 147 us, atomics queued on the few exponents; bisection with a vote per bit: 15.5 / 48 us.)
#include "common.h"
#include "spans.h"

namespace {

struct KeArgs {
    const char * mass, * pos, * n_used, * n_past;
    int64_t mass_nb2, mass_nb3, pos_nb2, pos_nb3;
    char * kept, * evicted;
    int64_t kept_nb2, kept_nb3, ev_nb2, ev_nb3;
    int n_kv, n_keep, n_evict, n_sink, n_recent, n_head_kv;
};

constexpr uint32_t KE_PINNED = 0xff800001u;           // just above the image of +inf
static __device__ __forceinline__ uint32_t ke_key(float m, bool keep) {
    if (keep) return KE_PINNED;
    if (m != m) m = -INFINITY;
    if (m == 0.0f) m = 0.0f;                          // -0 and +0 are equal
    const uint32_t u = __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int KE_BINS = 2048;

// reductions and prefix sums over a wave with DPP moves inside rows of 16 lanes and v_readlane between them (a ds_bpermute costs ~100 clocks)
template <int CTRL> static __device__ __forceinline__ uint32_t ke_dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <class OP> static __device__ __forceinline__ uint32_t ke_reduce(uint32_t v, OP op) {
    v = op(v, ke_dpp<0xB1>(v));      // quad_perm [1,0,3,2]
    v = op(v, ke_dpp<0x4E>(v));      // quad_perm [2,3,0,1]
    v = op(v, ke_dpp<0x141>(v));     // row_half_mirror
    v = op(v, ke_dpp<0x140>(v));     // row_mirror
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16), c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return op(op(a, b), op(c, d));
}
static __device__ __forceinline__ uint32_t ke_scan(uint32_t v) {      // inclusive prefix sum
    v += ke_dpp<0x111>(v);           // row_shr:1 .. 8, zeros shifted in
    v += ke_dpp<0x112>(v);
    v += ke_dpp<0x114>(v);
    v += ke_dpp<0x118>(v);
    const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31), c = b + __builtin_amdgcn_readlane(v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

// Wave w holds the slots from 64 C w on, lane by lane, C slots a lane: slot order is (wave, i, lane).  KPT > 0: C = KPT, keys in registers;
// KPT == 0: C from the length, keys read at every use.
template <int KPT, int NW>
__global__ void __launch_bounds__(64 * NW)
kv_select_kernel(const KeArgs a) {
    constexpr int NT = 64 * NW, PER = KE_BINS / NT;
    __shared__ __attribute__((aligned(16))) uint32_t hist[KE_BINS];
    __shared__ uint32_t lim[3][NW], part[NW], pick[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hk = blockIdx.x, i3 = blockIdx.y;
    const float * mass = (const float *)(a.mass + hk * a.mass_nb2 + i3 * a.mass_nb3);
    const int32_t * pos = (const int32_t *)(a.pos + hk * a.pos_nb2 + i3 * a.pos_nb3);
    int32_t * kept = (int32_t *)(a.kept + hk * a.kept_nb2 + i3 * a.kept_nb3);
    int32_t * evicted = a.evicted ? (int32_t *)(a.evicted + hk * a.ev_nb2 + i3 * a.ev_nb3) : nullptr;
    const int C = KPT > 0 ? KPT : (a.n_kv + NT - 1) / NT, first = wave * 64 * C + lane;
    float m[KPT > 0 ? KPT : 1]; int p[KPT > 0 ? KPT : 1];
    if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const int j = first + 64 * i;
            m[i] = j < a.n_kv ? mass[j] : 0.0f;
            p[i] = j < a.n_kv ? pos[j] : 0;
        }
    }
    int n = a.n_used ? ((const int32_t *)a.n_used)[i3] : a.n_kv;
    n = n < 0 ? 0 : n < a.n_kv ? n : a.n_kv;
    const int64_t recent = (int64_t)((const int32_t *)a.n_past)[i3] - a.n_recent;
    uint32_t key[KPT > 0 ? KPT : 1];                  // 0: not in use (below the image of -inf)
    if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) key[i] = first + 64 * i < n ? ke_key(m[i], p[i] < a.n_sink || p[i] >= recent) : 0;
    }
    auto each = [&](auto f) {                         // f(slot, key), in slot order within the wave, by all lanes
        if constexpr (KPT > 0) {
#pragma unroll
            for (int i = 0; i < KPT; i++) f(first + 64 * i, key[i]);
        } else {
            for (int i = 0; i < C; i++) {
                const int j = first + 64 * i;
                uint32_t k = 0;
                if (j < n) { const int q = pos[j]; k = ke_key(mass[j], q < a.n_sink || q >= recent); }
                f(j, k);
            }
        }
    };

    uint32_t T = 1;                                   // kept: key >= T, of which those equal to T only the first `equal`
    uint32_t equal = 0xffffffffu;
    if (n > a.n_keep) {
        // the range of the keys, the pinned ones counted aside
        uint32_t lo = 0xffffffffu, hi = 0, pinned = 0;
        each([&](int, uint32_t k) {
            if (k == KE_PINNED) pinned++;
            else if (k) { lo = lo < k ? lo : k; hi = hi > k ? hi : k; }
        });
        lo = ke_reduce(lo, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
        hi = ke_reduce(hi, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
        pinned = ke_reduce(pinned, [](uint32_t x, uint32_t y) { return x + y; });
        if (tid == 0) pick[3] = 0;
        if (lane == 0) { lim[0][wave] = lo; lim[1][wave] = hi; lim[2][wave] = pinned; }
        for (int i = tid; i < KE_BINS; i += NT) hist[i] = 0;
        __syncthreads();
        pinned = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) { lo = lo < lim[0][w] ? lo : lim[0][w]; hi = hi > lim[1][w] ? hi : lim[1][w]; pinned += lim[2][w]; }
        lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi); pinned = __builtin_amdgcn_readfirstlane(pinned);
        if (pinned >= (uint32_t)a.n_keep) { T = KE_PINNED; equal = a.n_keep; }
        else {
            uint32_t want = a.n_keep - pinned;          // rank of the wanted key among those in [lo, hi], from the largest
            for (;;) {
                const int bits = 32 - __builtin_clz((hi - lo) | 1), shift = bits > 11 ? bits - 11 : 0;
                each([&](int, uint32_t k) {
                    const bool in = k >= lo && k <= hi;
                    const uint32_t bin = (k - lo) >> shift;
                    const uint64_t who = __ballot(in);
                    if (!who) return;
                    const uint32_t one = __builtin_amdgcn_readlane(bin, __builtin_ctzll(who));
                    if (__ballot(in && bin == one) == who) { if (lane == 0) atomicAdd(&hist[one], (uint32_t)__popcll(who)); }
                    else if (in) atomicAdd(&hist[bin], 1u);
                });
                __syncthreads();
                // thread t owns the bins from the top down: PER (t + 1) - 1 .. PER t counted from the highest
                uint32_t h[PER], sum = 0;
#pragma unroll
                for (int i = 0; i < PER; i++) { h[i] = hist[KE_BINS - 1 - (tid * PER + i)]; sum += h[i]; }
                const uint32_t incl = ke_scan(sum);
                if (lane == 63) part[wave] = incl;
                __syncthreads();                      // (every bin has been read)
                uint32_t above = incl - sum;
#pragma unroll
                for (int w = 0; w < NW; w++) above += w < wave ? part[w] : 0;
                if (above < want && want <= above + sum) {
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        if (above < want && want <= above + h[i]) { pick[0] = KE_BINS - 1 - (tid * PER + i); pick[1] = want - above; pick[2] = h[i]; }
                        above += h[i];
                    }
                }
                for (int i = tid; i < KE_BINS; i += NT) hist[i] = 0;
                __syncthreads();
                const uint32_t bin = pick[0], in_bin = pick[2];
                want = pick[1];
                lo += bin << shift;
                if (shift == 0 || want == in_bin) { T = lo; if (want != in_bin) equal = want; break; }
                const uint32_t top = lo + ((1u << shift) - 1);
                hi = top < hi ? top : hi;
                if (in_bin <= 128) {                  // few are left: a thread each ranks them against one another (a pass more costs 1.5 us)
                    each([&](int, uint32_t k) { if (k >= lo && k <= hi) hist[atomicAdd(&pick[3], 1u)] = k; });
                    __syncthreads();
                    if (tid < (int)in_bin) {
                        const uint32_t k = hist[tid];
                        uint32_t over = 0, same = 0;
                        for (uint32_t i = 0; i < in_bin; i += 4) {      // (cells past the last hold 0)
                            const v4i x = *(const v4i *)&hist[i];
#pragma unroll
                            for (int q = 0; q < 4; q++) { over += (uint32_t)x[q] > k; same += (uint32_t)x[q] == k; }
                        }
                        if (over < want && want <= over + same) { pick[0] = k; pick[1] = want - over; pick[2] = same; }   // (every equal writes the same)
                    }
                    __syncthreads();
                    T = pick[0];
                    if (pick[1] != pick[2]) equal = pick[1];
                    break;
                }
            }
        }
        T = __builtin_amdgcn_readfirstlane(T); equal = __builtin_amdgcn_readfirstlane(equal);
    }
    // the wave's equals (where not all are kept) and kept ones before it, then each slot's own rank
    uint32_t eq_before = 0;
    const bool ties = equal != 0xffffffffu;
    const uint64_t below = (1ull << lane) - 1;
    if (ties) {
        uint32_t eq = 0;
        each([&](int, uint32_t k) { eq += __popcll(__ballot(k == T)); });
        __syncthreads();                              // (part has been read)
        if (lane == 0) part[wave] = eq;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) eq_before += w < wave ? part[w] : 0;
    }
    uint32_t e = eq_before;
    auto stays = [&](uint32_t k) {                    // the kept lanes at one i; called for i = 0, 1, ... in turn
        if (!ties) return (uint64_t)__ballot(k >= T);
        const uint64_t be = __ballot(k == T);
        const uint64_t b = __ballot(k > T || (k == T && e + __popcll(be & below) < equal));
        e += __popcll(be);
        return b;
    };
    int mine = 0;
    each([&](int, uint32_t k) { mine += __popcll(stays(k)); });
    if (lane == 0) lim[0][wave] = mine;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) { before += w < wave ? lim[0][w] : 0; all += lim[0][w]; }
    e = eq_before;
    each([&](int j, uint32_t k) {
        const uint64_t b = stays(k);
        const int rank = before + __popcll(b & below);
        if (b >> lane & 1) kept[rank] = j;
        else if (j < n && evicted && j - rank < a.n_evict) evicted[j - rank] = j;      // (j - rank slots before j are not kept)
        before += __popcll(b);
    });
    for (int j = all + tid; j < a.n_keep; j += NT) kept[j] = -1;
    if (evicted) for (int j = n - all + tid; j < a.n_evict; j += NT) evicted[j] = -1;
}

struct KgArgs {
    const char * kept;
    int64_t kept_nb2, kept_nb3;
    const char * src[2]; char * dst[2];
    int64_t s_nb1[2], s_nb2[2], s_nb3[2], d_nb1[2], d_nb2[2], d_nb3[2];
    int row_bytes[2], n_keep;
    const char * mass, * pos;
    int64_t mass_nb2, mass_nb3, pos_nb2, pos_nb3;
    char * mass_out, * pos_out;
    int64_t mo_nb2, mo_nb3, po_nb2, po_nb3;
};

// A group of W lanes (a power of two, the pieces of a row rounded up) copies a row; a workgroup takes 4 groups' worth of rows per thread, whose
// loads are all requested before the first is stored.  Bound by the rows' bytes, once in and once out.
template <class PIECE>
__global__ void __launch_bounds__(256)
kv_gather_kernel(const KgArgs a, int log2_w) {
    const int hk = blockIdx.y, i3 = blockIdx.z, lane = threadIdx.x & ((1 << log2_w) - 1), rows = 256 >> log2_w;
    const int32_t * kept = (const int32_t *)(a.kept + hk * a.kept_nb2 + i3 * a.kept_nb3);
    const char * src[2] = {a.src[0] + hk * a.s_nb2[0] + i3 * a.s_nb3[0], a.src[1] + hk * a.s_nb2[1] + i3 * a.s_nb3[1]};
    char * dst[2] = {a.dst[0] + hk * a.d_nb2[0] + i3 * a.d_nb3[0], a.dst[1] + hk * a.d_nb2[1] + i3 * a.d_nb3[1]};
    int i[4], j[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
        i[u] = blockIdx.x * 4 * rows + u * rows + ((int)threadIdx.x >> log2_w);
        j[u] = i[u] < a.n_keep ? kept[i[u]] : -1;
    }
    if (lane == 0) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (i[u] >= a.n_keep) continue;
            if (a.mass_out) ((float *)(a.mass_out + hk * a.mo_nb2 + i3 * a.mo_nb3))[i[u]] = j[u] < 0 ? 0.0f : ((const float *)(a.mass + hk * a.mass_nb2 + i3 * a.mass_nb3))[j[u]];
            if (a.pos_out) ((int32_t *)(a.pos_out + hk * a.po_nb2 + i3 * a.po_nb3))[i[u]] = j[u] < 0 ? -1 : ((const int32_t *)(a.pos + hk * a.pos_nb2 + i3 * a.pos_nb3))[j[u]];
        }
    }
    for (int e = lane; e * (int)sizeof(PIECE) < (a.row_bytes[0] > a.row_bytes[1] ? a.row_bytes[0] : a.row_bytes[1]); e += 1 << log2_w) {
        PIECE x[2][4];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int u = 0; u < 4; u++) if (j[u] >= 0 && e * (int)sizeof(PIECE) < a.row_bytes[s]) x[s][u] = *(const PIECE *)(src[s] + j[u] * a.s_nb1[s] + e * (int)sizeof(PIECE));
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int u = 0; u < 4; u++) if (j[u] >= 0 && e * (int)sizeof(PIECE) < a.row_bytes[s]) *(PIECE *)(dst[s] + i[u] * a.d_nb1[s] + e * (int)sizeof(PIECE)) = x[s][u];
    }
}

template <class PIECE> static int gather_launch(const KgArgs & g, int64_t n_keep, int64_t hk, int64_t ne3, hipStream_t s) {
    const int bytes = g.row_bytes[0] > g.row_bytes[1] ? g.row_bytes[0] : g.row_bytes[1], pieces = bytes / (int)sizeof(PIECE);
    int w = 0;
    while (w < 6 && (1 << w) < pieces) w++;
    const int64_t rows = 4 * (256 >> w);
    MI355_LAUNCH("kv_gather", kv_gather_kernel<PIECE>, dim3((unsigned)((n_keep + rows - 1) / rows), (unsigned)hk, (unsigned)ne3), dim3(256), 0, s, g, w);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
template <int KPT, int NW> static int select_launch(const KeArgs & a, int64_t ne3, hipStream_t s) {
    MI355_LAUNCH("kv_select", (kv_select_kernel<KPT, NW>), dim3((unsigned)a.n_head_kv, (unsigned)ne3), dim3(64 * NW), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
static int select_dispatch(const KeArgs & a, int64_t ne3, hipStream_t s) {
    if (a.n_kv <= 1024)  return select_launch<4, 4>(a, ne3, s);
    if (a.n_kv <= 4096)  return select_launch<8, 8>(a, ne3, s);
    if (a.n_kv <= 8192)  return select_launch<8, 16>(a, ne3, s);
    if (a.n_kv <= 16384) return select_launch<16, 16>(a, ne3, s);
    if (a.n_kv <= 32768) return select_launch<32, 16>(a, ne3, s);
    return select_launch<0, 16>(a, ne3, s);
}

} // namespace

extern "C" {

int mi355_kv_evict(const mi355_kv_evict_args * p, void * stream) {
    // (tensors of no sequences or no slots have no address)
    if (!p || (p->ne3 != 0 && ((p->n_kv > 0 && (!p->mass || !p->slot_pos)) || !p->n_past || !p->kept))) return MI355_E_NULL;
    if (p->ne3 != 0 && p->n_kv > 0 && (!p->k != !p->k_out || !p->v != !p->v_out)) return MI355_E_NULL;
    constexpr int64_t most = 1 << 30;                 // (32-bit slot numbers, a workgroup's stride past the last)
    if (p->n_kv < 0 || p->n_kv > most || p->n_keep < 1 || p->n_keep > most || p->n_evict < 0 || p->n_evict > most) return MI355_E_SHAPE;
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
    // what is written lies apart from what is read, and each output from the others: a slot may be read after its place has been written
    const int64_t hk = p->n_head_kv, ne3 = p->ne3, placed = p->n_keep < p->n_kv ? p->n_keep : p->n_kv;
    const int64_t bk = p->k ? mi355_row_size(p->type_kv, p->d) : 0, bv = p->v ? mi355_row_size(p->type_kv, dv) : 0;
    const Span in[] = {{p->mass, p->n_kv * 4, 1, 0, hk, p->mass_nb2, ne3, p->mass_nb3}, {p->slot_pos, p->n_kv * 4, 1, 0, hk, p->pos_nb2, ne3, p->pos_nb3},
                       {p->n_used, ne3 * 4, 1, 0, 1, 0, 1, 0}, {p->n_past, ne3 * 4, 1, 0, 1, 0, 1, 0},
                       {p->k, bk, p->n_kv, p->k_nb1, hk, p->k_nb2, ne3, p->k_nb3}, {p->v, bv, p->n_kv, p->v_nb1, hk, p->v_nb2, ne3, p->v_nb3}};
    const Span out[] = {{p->kept, p->n_keep * 4, 1, 0, hk, p->kept_nb2, ne3, p->kept_nb3}, {p->evicted, p->n_evict * 4, 1, 0, hk, p->ev_nb2, ne3, p->ev_nb3},
                        {p->k_out, bk, placed, p->ko_nb1, hk, p->ko_nb2, ne3, p->ko_nb3}, {p->v_out, bv, placed, p->vo_nb1, hk, p->vo_nb2, ne3, p->vo_nb3},
                        {p->mass_out, p->n_keep * 4, 1, 0, hk, p->mo_nb2, ne3, p->mo_nb3}, {p->pos_out, p->n_keep * 4, 1, 0, hk, p->po_nb2, ne3, p->po_nb3}};
    if (ne3 > 0) for (const Span & o : out) {
        for (const Span & x : in) if (spans_meet(o, x)) return MI355_E_UNSUPPORTED;
        for (const Span * x = out; x != &o; x++) if (spans_meet(o, *x)) return MI355_E_UNSUPPORTED;
    }
    // a row of 64 pieces and more takes a wave, 16 of them a workgroup: a grid dimension's 2^32 threads hold 2^28 such rows
    if ((p->k || p->v) && p->n_keep >= 1 << 28) return MI355_E_SHAPE;
    if (ne3 > 0) for (const Span & o : out) if (o.folds()) return MI355_E_UNSUPPORTED;
    if (p->ne3 == 0) return MI355_OK;

    KeArgs a;
    a.mass = (const char *)p->mass; a.mass_nb2 = p->mass_nb2; a.mass_nb3 = p->mass_nb3;
    a.pos = (const char *)p->slot_pos; a.pos_nb2 = p->pos_nb2; a.pos_nb3 = p->pos_nb3;
    a.n_used = (const char *)p->n_used; a.n_past = (const char *)p->n_past;
    a.kept = (char *)p->kept; a.kept_nb2 = p->kept_nb2; a.kept_nb3 = p->kept_nb3;
    a.evicted = (char *)p->evicted; a.ev_nb2 = p->ev_nb2; a.ev_nb3 = p->ev_nb3;
    a.n_kv = (int)p->n_kv; a.n_keep = (int)p->n_keep; a.n_evict = (int)p->n_evict; a.n_sink = p->n_sink; a.n_recent = p->n_recent; a.n_head_kv = (int)p->n_head_kv;
    hipStream_t s = (hipStream_t)stream;
    const int rc = select_dispatch(a, p->ne3, s);
    if (rc != MI355_OK) return rc;
    if (!p->k && !p->v && !p->mass_out && !p->pos_out) return MI355_OK;

    KgArgs g;
    g.kept = a.kept; g.kept_nb2 = a.kept_nb2; g.kept_nb3 = a.kept_nb3;
    g.src[0] = (const char *)p->k; g.s_nb1[0] = p->k_nb1; g.s_nb2[0] = p->k_nb2; g.s_nb3[0] = p->k_nb3;
    g.dst[0] = (char *)p->k_out; g.d_nb1[0] = p->ko_nb1; g.d_nb2[0] = p->ko_nb2; g.d_nb3[0] = p->ko_nb3;
    g.src[1] = (const char *)p->v; g.s_nb1[1] = p->v_nb1; g.s_nb2[1] = p->v_nb2; g.s_nb3[1] = p->v_nb3;
    g.dst[1] = (char *)p->v_out; g.d_nb1[1] = p->vo_nb1; g.d_nb2[1] = p->vo_nb2; g.d_nb3[1] = p->vo_nb3;
    g.row_bytes[0] = (int)bk; g.row_bytes[1] = (int)bv;
    g.n_keep = a.n_keep;
    g.mass = a.mass; g.mass_nb2 = a.mass_nb2; g.mass_nb3 = a.mass_nb3; g.pos = a.pos; g.pos_nb2 = a.pos_nb2; g.pos_nb3 = a.pos_nb3;
    g.mass_out = (char *)p->mass_out; g.mo_nb2 = p->mo_nb2; g.mo_nb3 = p->mo_nb3;
    g.pos_out = (char *)p->pos_out; g.po_nb2 = p->po_nb2; g.po_nb3 = p->po_nb3;
    // the widest piece that rows, strides and row lengths allow
    int64_t low = rows;
    if (p->k) low |= g.row_bytes[0];
    if (p->v) low |= g.row_bytes[1];
    if ((low & 15) == 0) return gather_launch<v4i>(g, p->n_keep, p->n_head_kv, p->ne3, s);
    if ((low & 7) == 0)  return gather_launch<v2i>(g, p->n_keep, p->n_head_kv, p->ne3, s);
    if ((low & 3) == 0)  return gather_launch<uint32_t>(g, p->n_keep, p->n_head_kv, p->ne3, s);
    return gather_launch<uint16_t>(g, p->n_keep, p->n_head_kv, p->ne3, s);
}

} // extern "C"
