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
    const char * k; uint32_t k_nb1; int64_t k_nb2, k_nb3;        // (rows at most 2 GiB apart: a row's address is one 32 x 32 + 64 bit multiply-add)
    const char * v; uint32_t v_nb1; int64_t v_nb2, v_nb3;
    const char * mask; int64_t m_nb1, m_nb2, m_nb3; int m_ne2, m_ne3;
    char * dst; int64_t d_nb1, d_nb2, d_nb3;
    const char * mass_in; int64_t in_nb2, in_nb3;
    char * mass_out; int64_t out_nb2, out_nb3;
    int n_q, n_kv, n_head, n_head_kv, d, dv;
    float scale, max_bias, logit_softcap, m0, m1, decay;
    uint32_t n_head_log2;
    int ratio; uint32_t by_ratio;   // heads per KV head; ceil(2^32 / ratio), 0 for ratio 1 (r / ratio without a division)
    int nsplit, lpitch;
    float * logits;     // steps: [ne3][n_head_kv][rows][lpitch], log2 domain
    float * stats;      // steps: [ne3][n_head_kv][nsplit][rows][2]: maximum (log2 domain) and sum; prompts: [ne3][n_head][n_q][2]: m, 1 / l
    float * part;       // steps: [ne3][n_head_kv][nsplit][rows][D]
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

// row r of a KV head = (query, head of the group); r < 2^16
static __device__ __forceinline__ int m_query(const MArgs & a, int r) { return a.by_ratio ? (int)__umulhi((uint32_t)r, a.by_ratio) : r; }
static __device__ __forceinline__ const char * m_mask(const MArgs & a, int iq, int h, int i3) {
    return a.mask + iq * a.m_nb1 + (a.m_ne2 > 1 ? h % a.m_ne2 : 0) * a.m_nb2 + (a.m_ne3 > 1 ? i3 % a.m_ne3 : 0) * a.m_nb3;
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

// ---- decode steps (at most 8 queries): one pass over K and V on the matrix cores --------------------------------------------------------
//
// Bound by the cache's bytes: at GQA 4..8 the rows that meet a K or V row fill one 16-row matrix tile, so the arithmetic is small change.
// A wave owns 32 slots at a time, nothing is shared between waves until the end:
//   S^T[slot][row] = K Q^T      v_mfma_f32_16x16x32: K rows come from memory straight into the A operand (lane = slot, 16 bytes each)
//   O^T[f][row]   += V^T P^T    P^T is the S^T accumulator as it lies; V goes through LDS and is read transposed (ds_read_b64_tr_b16)
// A "row" is a (query, head of the KV head) pair.  f32 results from 16-bit operands: q and P are split into two f16 (three bf16) parts whose
// products are added in the accumulator, 22 (24) bits; cache values are exact in 16 bits (blocks: their integers, scales applied in f32 --
// K's to the partial products of each 32-block, V's to P).  Logits are kept (log2 domain) for the pass that forms the weights.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;

template <int TYPE> struct Fmt {       // 16-bit format of the operands and the parts an f32 is split into
    static constexpr bool bf = TYPE == MI355_TYPE_BF16, quant = TYPE == MI355_TYPE_Q8_0 || TYPE == MI355_TYPE_Q4_0;
    static constexpr int parts = bf ? 3 : 2;
    static constexpr int block = TYPE == MI355_TYPE_Q8_0 ? 34 : 18;
};
template <bool BF> static __device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else              return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// x[8] -> parts of 8 16-bit values each, part 0 the largest.  f16: rounded, then the rest rounded; bf16: upper halves, cut off
template <bool BF, int P> static __device__ __forceinline__ void split8(const float * x, v4i * out) {
    if constexpr (BF) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t u0 = __float_as_uint(r[2 * i]), u1 = __float_as_uint(r[2 * i + 1]);
                out[p][i] = (int)__builtin_amdgcn_perm(u1, u0, 0x07060302u);
                r[2 * i] -= __uint_as_float(u0 & 0xffff0000u);
                r[2 * i + 1] -= __uint_as_float(u1 & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // one rounding of hi for both of its uses: left to itself the compiler folds the product behind x into the operand's conversion
            // (one rounding) but not into lo's (two), and near a tie lo then belongs to the other neighbour
            int bits = __builtin_bit_cast(int, h2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
            asm("" : "+v"(bits));
            const h2 hi = __builtin_bit_cast(h2, bits);
            const h2 lo = {(_Float16)__builtin_fmaf((float)hi[0], -1.0f, x[2 * i]), (_Float16)__builtin_fmaf((float)hi[1], -1.0f, x[2 * i + 1])};
            out[0][i] = bits;
            out[1][i] = __builtin_bit_cast(int, lo);
        }
    }
}

// 8 consecutive features (chunk j) of a cache row on their way to an operand: the bytes, then 16-bit values (blocks: the integers)
template <int TYPE> struct Chunk {
    v4i raw;
    static __device__ __forceinline__ int at(int j) { return j * 16; }       // byte offset of chunk j in a row
    __device__ __forceinline__ void load(const char * p) { raw = *(const v4i *)p; }
    __device__ __forceinline__ v4i operand(int) const { return raw; }
};
static __device__ __forceinline__ v4i bytes_f16(uint32_t w0, uint32_t w1, float bias) {      // 8 bytes -> f16 of (byte - bias); 0x6400 | b is 1024 + b
    const _Float16 c = (_Float16)(1024.0f + bias);
    const h2 cc = {c, c};
    v4i r;
    r[0] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) - cc);
    r[1] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) - cc);
    r[2] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) - cc);
    r[3] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) - cc);
    return r;
}
template <> struct Chunk<MI355_TYPE_Q8_0> {
    uint32_t w0, w1;
    static __device__ __forceinline__ int at(int j) { return (j >> 2) * 34 + 2 + (j & 3) * 8; }
    __device__ __forceinline__ void load(const char * p) { __builtin_memcpy(&w0, p, 4); __builtin_memcpy(&w1, p + 4, 4); }
    __device__ __forceinline__ v4i operand(int) const { return bytes_f16(w0 ^ 0x80808080u, w1 ^ 0x80808080u, 128.0f); }
};
template <> struct Chunk<MI355_TYPE_Q4_0> {
    uint32_t w0, w1;
    static __device__ __forceinline__ int at(int j) { return (j >> 2) * 18 + 2 + (j & 1) * 8; }
    __device__ __forceinline__ void load(const char * p) { __builtin_memcpy(&w0, p, 4); __builtin_memcpy(&w1, p + 4, 4); }
    __device__ __forceinline__ v4i operand(int j) const {
        const int sh = (j & 2) * 2;
        return bytes_f16((w0 >> sh) & 0x0f0f0f0fu, (w1 >> sh) & 0x0f0f0f0fu, 8.0f);
    }
};
// the same 8 bytes out of raw rows in LDS, whose words are what it reads: a block's integers start 2 bytes past a word in even blocks, on a
// word in odd ones (34 and 18 are 2 mod 4)
template <int TYPE> static __device__ __forceinline__ Chunk<TYPE> raw_chunk(const uint8_t * row, int j) {
    const bool odd = j >> 2 & 1;
    const uint32_t * q = (const uint32_t *)(row + Chunk<TYPE>::at(j) - (odd ? 4 : 2));
    const uint32_t x0 = q[0], x1 = q[1], x2 = q[2], pick = odd ? 0x07060504u : 0x05040302u;
    Chunk<TYPE> c;
    c.w0 = __builtin_amdgcn_perm(x1, x0, pick);
    c.w1 = __builtin_amdgcn_perm(x2, x1, pick);
    return c;
}
// non-finite 16-bit values of a chunk -> 0; true if there was one
template <bool BF> static __device__ __forceinline__ bool sanitize(v4i & x) {
    bool bad = false;
    constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t u = (uint32_t)x[i];
        if ((u & e) == e) { u &= 0xffff0000u; bad = true; }
        if ((u & (e << 16)) == (e << 16)) { u &= 0xffffu; bad = true; }
        x[i] = (int)u;
    }
    return bad;
}

static __device__ __forceinline__ float max_groups(float v) {       // over the four 16-lane groups, lanes of equal place
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
static __device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// RT: 16-row tiles of a workgroup.  RP (blocks only): the 16 columns of a tile are RP rows times 16 / RP classes of 32-blocks -- at GQA 4 or 8
// the columns that would repeat a row each scale P by the blocks of their class, so a lane forms D / 32 / (16 / RP) scaled copies of P and not
// D / 32; a feature tile takes its result from the columns of its block's class.
// RAW (blocks only, step_raw): rows come in as consecutive pieces of D / 16 bytes (17 or 9 a row) and are taken apart in LDS.  A lane that loads
// the 8 bytes of its own chunk reads at every second byte address, which the address unit serves a lane per clock: the 20 loads of a
// tile then cost a CU's 8 waves 4 us before the first product.
template <int TYPE, int D, int NW, bool HASV, int RT, int RP, bool RAW>
__global__ void __launch_bounds__(NW * 64, D <= 64 ? (RT == 1 ? 3 : 2) : D <= 128 ? 2 : 1)
mass_step_kernel(const MArgs a) {
    typedef Fmt<TYPE> F;
    static_assert(!RAW || F::quant, "raw rows are block rows");
    constexpr int KS = D / 32, FT = D / 16, P = F::parts;
    constexpr int NC = 16 / RP, SETS = KS > NC ? KS / NC : 1;   // classes of blocks, scaled copies of P per lane
    constexpr int VR = 512 / D, VN = D / 16;                    // V rows per 64 chunks, groups of 64 chunks of a tile
    constexpr int VP = D * 2 + 32;                              // V tile row pitch (bytes)
    constexpr int OP = D + 4;                                   // merge row pitch (floats)
    constexpr int VB = HASV ? (32 * VP > 16 * OP * 4 ? 32 * VP : 16 * OP * 4) : F::quant ? 32 * VP : 16;
    constexpr int DN = KS / 2;                                  // scales of a tile per lane: 32 rows x KS blocks over 64 lanes
    constexpr int PB = D / 16, PR = F::block / 2, PN = (32 * PR + 63) / 64;    // RAW: bytes of a piece, pieces of a row, pieces of a tile per lane
    typedef uint32_t piece_t __attribute__((ext_vector_type(PB / 4)));
    typedef _Float16 hk_t __attribute__((ext_vector_type(KS)));
    __shared__ __attribute__((aligned(16))) uint8_t lds[NW][VB];
    __shared__ v4i qs[RT][KS][P][64];
    uint8_t (&raw)[NW][VB] = lds;                               // RAW: raw rows of K, then of V, then V's values, one after the other
    static_assert(!RAW || VB >= 32 * PR * PB + 16, "raw rows fit");
    __shared__ __attribute__((aligned(16))) uint16_t kd[F::quant ? NW : 1][F::quant ? 32 * KS : 8], vd[F::quant && HASV ? NW : 1][F::quant && HASV ? 32 * KS : 8];
    __shared__ float wm[NW][16 * RT], wl[NW][16 * RT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const int ratio = a.ratio, R = ratio * a.n_q;
    const int hk = blockIdx.y, rb = blockIdx.x / a.nsplit * 16 * RT, i3 = blockIdx.z, split = blockIdx.x % a.nsplit;
    const char * kb = a.k + hk * a.k_nb2 + i3 * a.k_nb3;
    const char * vb = HASV ? a.v + hk * a.v_nb2 + i3 * a.v_nb3 : nullptr;
    const bool m8 = a.mask && (((uintptr_t)a.mask | (uintptr_t)a.m_nb1 | (uintptr_t)a.m_nb2 | (uintptr_t)a.m_nb3) & 7) == 0;
    const bool capped = a.logit_softcap != 0.0f;
    // this lane's rows (columns past the last one repeat it)
    int r[RT];
    const char * mrow[RT];
#pragma unroll
    for (int x = 0; x < RT; x++) {
        r[x] = rb + 16 * x + lr % RP;
        if (r[x] >= R) r[x] = R - 1;
        const int iq = m_query(a, r[x]), h = hk * ratio + r[x] - iq * ratio;
        mrow[x] = m_mask(a, iq, h, i3);
    }

    // chunks past the head size re-read the last one: they meet zeros of q, and features of V that are not stored.  Slots past the end re-read
    // the last one and are hidden
    const int ntiles = (a.n_kv + 31) / 32, TW = a.nsplit * NW;
    Chunk<TYPE> kc[F::quant ? 1 : 2][RAW ? 1 : F::quant ? VN : KS], vc[HASV && !RAW ? VN : 1];
    uint16_t ksc[F::quant && !RAW ? DN : 1], vsc[F::quant && !RAW && HASV ? DN : 1];
    piece_t kp[RAW ? PN : 1], vp[RAW && HASV ? PN : 1];
    uint32_t koff[RAW ? PN : 1], voff[RAW && HASV ? PN : 1];   // of this lane's pieces from a tile's first row
    const int vcc = lane % (D / 8) < a.dv / 8 ? lane % (D / 8) : a.dv / 8 - 1;
    const char * vl = vb + Chunk<TYPE>::at(vcc);
    const int kcc = lane % (D / 8) < a.d / 8 ? lane % (D / 8) : a.d / 8 - 1;
    const char * kl = kb + Chunk<TYPE>::at(kcc);
    if constexpr (RAW) {
#pragma unroll
        for (int i = 0; i < PN; i++) {
            const uint32_t n = 64 * i + lane < 32 * PR ? 64 * i + lane : 32 * PR - 1, row = n / PR;
            koff[i] = row * a.k_nb1 + (n - row * PR) * PB;
            if constexpr (HASV) voff[i] = row * a.v_nb1 + (n - row * PR) * PB;
        }
    }
    auto load_raw = [&](const char * base, uint32_t nb1, const uint32_t * off, int t, piece_t * out) {
        const char * tile = base + (uint64_t)(32u * (uint32_t)t) * nb1;
        if (32 * t + 32 <= a.n_kv) {
#pragma unroll
            for (int i = 0; i < PN; i++) out[i] = *(const piece_t *)(tile + off[i]);
        } else {
            const uint32_t last = a.n_kv - 1 - 32 * t;
#pragma unroll
            for (int i = 0; i < PN; i++) {
                const uint32_t n = 64 * i + lane < 32 * PR ? 64 * i + lane : 32 * PR - 1, row = n / PR;
                out[i] = *(const piece_t *)(tile + (row < last ? row : last) * nb1 + (n - row * PR) * PB);
            }
        }
    };
    auto put_raw = [&](const piece_t * in) {
#pragma unroll
        for (int i = 0; i < PN; i++) if (64 * i + 64 <= 32 * PR || 64 * i + lane < 32 * PR) *(piece_t *)(raw[wave] + (64 * i + lane) * PB) = in[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    auto raw_scales = [&](uint16_t * out) {
#pragma unroll
        for (int i = 0; i < DN; i++) { const int n = 64 * i + lane; out[n] = *(const uint16_t *)(raw[wave] + n / KS * PR * PB + n % KS * F::block); }
    };
    auto slot = [&](int j) { return (uint64_t)(uint32_t)(j < a.n_kv ? j : a.n_kv - 1); };
    auto load_scales = [&](const char * base, uint32_t nb1, int dim, int t, uint16_t * out) {
#pragma unroll
        for (int i = 0; i < DN; i++) {
            const int n = 64 * i + lane, b = n % KS < dim / 32 ? n % KS : dim / 32 - 1;
            out[i] = *(const uint16_t *)(base + slot(32 * t + n / KS) * nb1 + b * F::block);
        }
    };
    auto load_k = [&](int t) {
        if constexpr (RAW) load_raw(kb, a.k_nb1, koff, t, kp);
        else if constexpr (F::quant) {
#pragma unroll
            for (int i = 0; i < VN; i++) kc[0][i].load(kl + slot(32 * t + VR * i + lane / (D / 8)) * a.k_nb1);
            load_scales(kb, a.k_nb1, a.d, t, ksc);
        } else {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const char * row = kb + slot(32 * t + 16 * u + lr) * a.k_nb1;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) kc[u][ks].load(row + Chunk<TYPE>::at(4 * ks + g < a.d / 8 ? 4 * ks + g : a.d / 8 - 1));
            }
        }
    };
    auto load_v = [&](int t) {
        if constexpr (HASV && RAW) load_raw(vb, a.v_nb1, voff, t, vp);
        else if constexpr (HASV) {
#pragma unroll
            for (int i = 0; i < VN; i++) vc[i].load(vl + slot(32 * t + VR * i + lane / (D / 8)) * a.v_nb1);
            if constexpr (F::quant) load_scales(vb, a.v_nb1, a.dv, t, vsc);
        }
    };
    // mask of slots 32 t + 16 u + 4 g + i as it lies, -inf past the last slot
    auto load_mask = [&](int t, u2 (&w)[RT][2]) {
#pragma unroll
        for (int x = 0; x < RT; x++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int j = 32 * t + 16 * u + 4 * g;
                if (m8 && j + 4 <= a.n_kv) w[x][u] = *(const u2 *)(mrow[x] + 2 * (int64_t)j);
                else {
                    uint32_t y[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = j + i >= a.n_kv ? 0xfc00u : a.mask ? ((const uint16_t *)mrow[x])[j + i] : 0u;
                    w[x][u] = u2{y[0] | y[1] << 16, y[2] | y[3] << 16};
                }
            }
    };
    auto sees = [&](const u2 (&w)[RT][2]) {
        bool all = true;
#pragma unroll
        for (int x = 0; x < RT; x++) all &= w[x][0].x == 0xfc00fc00u && w[x][0].y == 0xfc00fc00u && w[x][1].x == 0xfc00fc00u && w[x][1].y == 0xfc00fc00u;
        return __any(!all);
    };

    // tiles are dealt to the waves of all slices in turn: sequences shorter than the range keep them all busy.  A tile hidden from every row
    // costs its mask, which runs one tile ahead of the rows; the first tile is fetched without asking: one round trip instead of two
    int t = split * NW + wave;
    u2 mk[RT][2], mkn[RT][2];
    if (t < ntiles) { load_k(t); load_v(t); load_mask(t, mk); }
    if (t + TW < ntiles) load_mask(t + TW, mkn);

    // q for all waves, in LDS as the B operand takes it: a wave splits the 32-feature chunks that fall to it.  Scale and log2(e) go on q; for f16
    // the row's largest value is brought to [2^14, 2^15) by a power of two that the logits get back (its small values then stay clear of the
    // subnormal range)
    constexpr int QN = (KS + NW - 1) / NW;
    float qe[RT], slope[RT], y[RT][QN][8];
#pragma unroll
    for (int x = 0; x < RT; x++) {
        const int iq = m_query(a, r[x]), h = hk * ratio + r[x] - iq * ratio;
        slope[x] = m_slope(a, h) * LOG2E;
        const float * qp = (const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3);
        const float sc = capped ? a.scale / a.logit_softcap : a.scale * LOG2E;
        float amax = 0.0f;
#pragma unroll
        for (int n = 0; n < QN; n++) {
            const int f = 32 * (wave + NW * n) + 8 * g;
            v4f y0 = {0.0f, 0.0f, 0.0f, 0.0f}, y1 = y0;
            if (f < a.d) { y0 = *(const v4f *)(qp + f) * sc; y1 = *(const v4f *)(qp + f + 4) * sc; }
#pragma unroll
            for (int i = 0; i < 4; i++) { y[x][n][i] = y0[i]; y[x][n][4 + i] = y1[i]; amax = fmaxf(amax, fmaxf(fabsf(y0[i]), fabsf(y1[i]))); }
        }
        if (!F::bf) {
            amax = max_groups(amax);
            if (g == 0) wm[wave][16 * x + lr] = amax;
        }
    }
    if (!F::bf) __syncthreads();
#pragma unroll
    for (int x = 0; x < RT; x++) {
        int e = 0;
        if (!F::bf) {
            float amax = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) amax = fmaxf(amax, wm[w][16 * x + lr]);
            e = amax > 0.0f && amax < INFINITY ? __builtin_amdgcn_frexp_expf(amax) - 15 : 0;
        }
        qe[x] = ldexpf(1.0f, e);
#pragma unroll
        for (int n = 0; n < QN; n++) {
            if (wave + NW * n >= KS) continue;
            v4i w[P];
#pragma unroll
            for (int i = 0; i < 8; i++) y[x][n][i] = ldexpf(y[x][n][i], -e);
            split8<F::bf, P>(y[x][n], w);
#pragma unroll
            for (int p = 0; p < P; p++) qs[x][wave + NW * n][p][lane] = w[p];
        }
    }
    __syncthreads();

    float m[RT], l[RT];                         // of this lane's rows; l over this lane's slots only
    int E[RT];                                  // blocks: o holds 2^(14 - E) times its value, E the exponent of the largest scale of V met so far
    v4f o[RT][HASV ? FT : 1];
    float * lg[RT];
#pragma unroll
    for (int x = 0; x < RT; x++) {
        m[x] = -INFINITY; l[x] = 0.0f; E[x] = -64;
#pragma unroll
        for (int i = 0; i < (HASV ? FT : 1); i++) o[x][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        lg[x] = a.logits + (((int64_t)i3 * a.n_head_kv + hk) * R + r[x]) * a.lpitch;
    }
    auto mine = [&](int x) { return lr < RP && rb + 16 * x + lr < R; };      // the lane that stores row r[x]

    while (t < ntiles) {
        u2 mc[RT][2];
#pragma unroll
        for (int x = 0; x < RT; x++) { mc[x][0] = mk[x][0]; mc[x][1] = mk[x][1]; }
        int tn = t + TW;                        // the next tile that a row sees
        while (tn < ntiles && !sees(mkn)) {
#pragma unroll
            for (int x = 0; x < RT; x++)
                if (mine(x)) {
#pragma unroll
                    for (int u = 0; u < 2; u++) if (32 * tn + 16 * u + 4 * g < a.lpitch) *(v4f *)(lg[x] + 32 * tn + 16 * u + 4 * g) = v4f{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                }
            tn += TW;
            if (tn < ntiles) load_mask(tn, mkn);
        }
        const bool next = tn < ntiles;
#pragma unroll
        for (int x = 0; x < RT; x++) { mk[x][0] = mkn[x][0]; mk[x][1] = mkn[x][1]; }
        if constexpr (RAW) { put_raw(kp); raw_scales(kd[wave]); __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
        else if constexpr (F::quant) {          // K's integers to rows, the scales of the 32 slots where every lane can read them
#pragma unroll
            for (int i = 0; i < VN; i++) *(v4i *)(lds[wave] + (VR * i + lane / (D / 8)) * VP + lane % (D / 8) * 16) = kc[0][i].operand(kcc);
#pragma unroll
            for (int i = 0; i < DN; i++) {
                kd[wave][64 * i + lane] = ksc[i];
                if constexpr (HASV) vd[wave][64 * i + lane] = vsc[i];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        // ---- S^T
        v4f c[RT][2];
        {
            hk_t dk[2][4];
            if constexpr (F::quant) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) dk[u][i] = *(const hk_t *)&kd[wave][(16 * u + 4 * g + i) * KS];
            }
#pragma unroll
            for (int x = 0; x < RT; x++) c[x][0] = c[x][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                v4i qv[RT][P];
#pragma unroll
                for (int x = 0; x < RT; x++)
#pragma unroll
                    for (int p = 0; p < P; p++) qv[x][p] = qs[x][ks][p][lane];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    v4i kop;
                    if constexpr (RAW) kop = raw_chunk<TYPE>(raw[wave] + (16 * u + lr) * PR * PB, 4 * ks + g).operand(g);
                    else if constexpr (F::quant) kop = *(const v4i *)(lds[wave] + (16 * u + lr) * VP + (4 * ks + g) * 16);
                    else kop = kc[u][ks].operand(g);
#pragma unroll
                    for (int x = 0; x < RT; x++) {
                        v4f b = F::quant ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : c[x][u];
#pragma unroll
                        for (int p = P - 1; p >= 0; p--) b = mfma16<F::bf>(kop, qv[x][p], b);
                        if constexpr (F::quant) {
#pragma unroll
                            for (int i = 0; i < 4; i++) c[x][u][i] = __builtin_fmaf(b[i], (float)dk[u][i][ks], c[x][u][i]);
                        } else c[x][u] = b;
                    }
                }
            }
        }
        if (next) load_k(tn);                   // in flight during the rest of this tile
        if (tn + TW < ntiles) load_mask(tn + TW, mkn);
        float s[RT][8], p[RT][8], corr[RT];     // slots 32 t + 16 (i >> 2) + 4 g + (i & 3)
        bool some = false;                      // some row does not see some slot of the tile
#pragma unroll
        for (int x = 0; x < RT; x++) {
            float mx = m[x];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float mv = h2f((uint16_t)(mc[x][i >> 2][(i & 3) >> 1] >> (16 * (i & 1))));
                float y = c[x][i >> 2][i & 3] * qe[x];
                if (capped) y = a.logit_softcap * LOG2E * tanhf(y);
                s[x][i] = mv == -INFINITY ? -INFINITY : __builtin_fmaf(mv, slope[x], y);
                mx = fmaxf(mx, s[x][i]);
                some |= s[x][i] == -INFINITY;
            }
            if (mine(x)) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int j = 32 * t + 16 * u + 4 * g;
                    if (j < a.lpitch) *(v4f *)(lg[x] + j) = v4f{s[x][4 * u], s[x][4 * u + 1], s[x][4 * u + 2], s[x][4 * u + 3]};
                }
            }
            mx = max_groups(mx);
            const float ms = mx == -INFINITY ? 0.0f : mx;
            corr[x] = __builtin_amdgcn_exp2f(m[x] - ms);        // m = -inf: 0
            l[x] *= corr[x];
#pragma unroll
            for (int i = 0; i < 8; i++) { p[x][i] = __builtin_amdgcn_exp2f(s[x][i] - ms); l[x] += p[x][i]; }
            m[x] = mx;
        }
        if constexpr (HASV) {
            const bool hidden = __any(some);
            _Float16 dd[RT][SETS][8];
            if constexpr (RAW) { put_raw(vp); raw_scales(vd[wave]); __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
            if constexpr (F::quant) {
                // the scales of V go on P, those of this lane's class of blocks.  A hidden slot's is taken as 0 (it may be NaN)
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    _Float16 dm = 0;
#pragma unroll
                    for (int q = 0; q < SETS; q++)
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int b = q * NC + lr / RP;
                            dd[x][q][i] = __builtin_bit_cast(_Float16, vd[wave][(16 * (i >> 2) + 4 * g + (i & 3)) * KS + (b < KS ? b : 0)]);
                        }
                    if (hidden) {
#pragma unroll
                        for (int q = 0; q < SETS; q++)
#pragma unroll
                            for (int i = 0; i < 8; i++) if (s[x][i] == -INFINITY) dd[x][q][i] = 0;
                    }
#pragma unroll
                    for (int q = 0; q < SETS; q++)
#pragma unroll
                        for (int i = 0; i < 8; i++) dm = __builtin_elementwise_max(dm, __builtin_elementwise_abs(dd[x][q][i]));
                    const float dmx = max_groups((float)dm);
                    const int e = dmx > 0.0f && dmx < INFINITY ? __builtin_amdgcn_frexp_expf(dmx) - 1 : -64;
                    const int En = E[x] > e ? E[x] : e;
                    corr[x] = ldexpf(corr[x], E[x] - En);
                    E[x] = En;
                }
            }
#pragma unroll
            for (int x = 0; x < RT; x++)
                if (__any(corr[x] != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < FT; i++) o[x][i] = o[x][i] * corr[x];
                }
            // ---- V tile into LDS.  A slot that some row does not see must not reach that row through 0 * NaN: its non-finite values are
            // taken out here and added below to the rows that do see it
            uint32_t bad = 0;                                   // slots of the tile with values taken out
            if constexpr (!F::quant) if (hidden) {
                uint32_t unseen = 0;                            // bit j: slot 32 t + j is hidden from some row
#pragma unroll
                for (int x = 0; x < RT; x++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint64_t b = __ballot(s[x][i] == -INFINITY);
#pragma unroll
                        for (int gg = 0; gg < 4; gg++) if ((b >> (16 * gg)) & 0xffff) unseen |= 1u << (16 * (i >> 2) + 4 * gg + (i & 3));
                    }
#pragma unroll
                for (int i = 0; i < VN; i++) {
                    const int row = VR * i + lane / (D / 8);
                    bool taken = false;
                    if (unseen >> row & 1) taken = sanitize<F::bf>(vc[i].raw);
                    const uint64_t b = __ballot(taken);
                    if (b) {
#pragma unroll
                        for (int q = 0; q < VR; q++) if (b >> (q * (D / 8)) & ((1ull << (D / 8)) - 1)) bad |= 1u << (i * VR + q);
                    }
                }
            }
            v4i vt16[VN];
#pragma unroll
            for (int i = 0; i < VN; i++) {
                if constexpr (RAW) vt16[i] = raw_chunk<TYPE>(raw[wave] + (VR * i + lane / (D / 8)) * PR * PB, vcc).operand(vcc);
                else vt16[i] = vc[i].operand(vcc);
            }
            if constexpr (RAW) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = 0; i < VN; i++) *(v4i *)(lds[wave] + (VR * i + lane / (D / 8)) * VP + lane % (D / 8) * 16) = vt16[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (next) load_v(tn);
            // ---- O^T
            const uint8_t * vt = lds[wave] + (4 * g + (lr >> 2)) * VP + 8 * (lr & 3);
            v4i pf[RT][P];
#pragma unroll
            for (int x = 0; x < RT; x++) {
                if constexpr (!F::bf) {                         // f16 parts: clear of the subnormal range
                    const float up = F::quant ? ldexpf(1.0f, 14 - E[x]) : 16384.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) p[x][i] *= up;
                }
                if constexpr (!F::quant) split8<F::bf, P>(p[x], pf[x]);
            }
#pragma unroll
            for (int f = 0; f < FT; f++) {
                if constexpr (F::quant) {
                    if (f % (FT / SETS) == 0) {                 // the next scaled copy
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            float y[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) y[i] = p[x][i] * (float)dd[x][f / (FT / SETS)][i];
                            split8<false, 2>(y, pf[x]);
                        }
                    }
                }
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(vt + 32 * f));
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(vt + 32 * f + 16 * VP));
                v4i vop;
                __builtin_memcpy(&vop, &lo, 8);
                __builtin_memcpy((char *)&vop + 8, &hi, 8);
#pragma unroll
                for (int x = 0; x < RT; x++)
#pragma unroll
                    for (int q = P - 1; q >= 0; q--) o[x][f] = mfma16<F::bf>(vop, pf[x][q], o[x][f]);
            }
            if (!F::quant && bad) {                             // non-finite values of slots that only some rows see
                for (int row = 0; row < 32; row++) {
                    if (!(bad >> row & 1)) continue;
                    const int from = ((row & 15) >> 2) * 16 + lr, i = (row >> 4) * 4 + (row & 3), j = 32 * t + row;
                    if (j >= a.n_kv) continue;
                    const char * vr = vb + (uint64_t)(uint32_t)j * a.v_nb1;
#pragma unroll
                    for (int x = 0; x < RT; x++) {
                        float pr = 0.0f, sr = -INFINITY;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            const float a0 = __shfl(p[x][q], from, 64), a1 = __shfl(s[x][q], from, 64);
                            if (q == i) { pr = a0; sr = a1; }
                        }
#pragma unroll
                        for (int f = 0; f < FT; f++)
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const int e = 16 * f + 4 * g + q;
                                if (e >= a.dv) continue;
                                const float y = kv_value<TYPE>(vr, e);
                                if (sr != -INFINITY && !(fabsf(y) < INFINITY)) o[x][f][q] += pr * y;
                            }
                    }
                }
            }
        }
        t = tn;
    }
    // ---- the waves' states meet in LDS
#pragma unroll
    for (int x = 0; x < RT; x++) {
        l[x] = sum_groups(l[x]);
        if (g == 0 && lr < RP) { wm[wave][16 * x + lr] = m[x]; wl[wave][16 * x + lr] = l[x]; }
    }
    const int64_t base = (((int64_t)i3 * a.n_head_kv + hk) * a.nsplit + split) * R + rb;
#pragma unroll
    for (int x = 0; x < RT; x++) {
        const int rows = R - rb - 16 * x < RP ? R - rb - 16 * x : RP;
        if constexpr (HASV) {
            if (x > 0) __syncthreads();                         // the tile before this one has been read
            float * ob = (float *)lds[wave] + lr % RP * OP + 4 * g;
            const float back = F::bf ? 1.0f : F::quant ? ldexpf(1.0f, E[x] - 14) : 1.0f / 16384.0f;
#pragma unroll
            for (int f = 0; f < FT; f++) if (NC == 1 || f / 2 % NC == lr / RP) *(v4f *)(ob + 16 * f) = o[x][f] * back;
        }
        __syncthreads();
        if constexpr (HASV) {
            for (int idx = tid; idx < rows * (D / 4); idx += NW * 64) {
                const int rr = idx / (D / 4), f4 = idx % (D / 4);
                if (4 * f4 >= a.dv) continue;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][16 * x + rr]);
                const float ms = M == -INFINITY ? 0.0f : M;
                v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < NW; w++) O = O + *(const v4f *)((const float *)lds[w] + rr * OP + 4 * f4) * __builtin_amdgcn_exp2f(wm[w][16 * x + rr] - ms);
                *(v4f *)(a.part + (base + 16 * x + rr) * D + 4 * f4) = O;
            }
        }
        if (tid < rows) {
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][16 * x + tid]);
            const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < NW; w++) L = __builtin_fmaf(wl[w][16 * x + tid], __builtin_amdgcn_exp2f(wm[w][16 * x + tid] - ms), L);
            *(v2f *)(a.stats + (base + 16 * x + tid) * 2) = v2f{M, L};
        }
    }
}

// The slices' statistics meet: workgroups 0 .. mass_wgs - 1 form the weights of 256 slots each from the logits, the others a row of dst each.
// Both start with loads that nothing precedes (a slice's statistics: one load per thread at 64 slices of 4 rows), so the launch is two
// memory round trips long.
template <int D>
__global__ void __launch_bounds__(256)
mass_finish_kernel(const MArgs a, int mass_wgs) {
    __shared__ float sm[256], sl[256];
    const int tid = threadIdx.x, hk = blockIdx.y, i3 = blockIdx.z;
    const int ratio = a.ratio, R = ratio * a.n_q;
    const int64_t base = ((int64_t)i3 * a.n_head_kv + hk) * a.nsplit * R;
    const v2f * st = (const v2f *)a.stats + base;
    if ((int)blockIdx.x < mass_wgs) {
        int w = 4;                                              // threads per row: 64 for up to 4 rows .. 4 for 64
        while (w < 64 && w * 2 * R <= 256) w *= 2;
        const int rows = 256 / w, j = blockIdx.x * 256 + tid;
        const float * lg = a.logits + ((int64_t)i3 * a.n_head_kv + hk) * R * a.lpitch + j;
        float t = 0.0f;
        for (int r0 = 0; r0 < R; r0 += rows) {
            float s4[4];                                        // the first logits, requested beside the statistics
#pragma unroll
            for (int i = 0; i < 4; i++) s4[i] = j < a.n_kv && r0 + i < R ? lg[(int64_t)(r0 + i) * a.lpitch] : -INFINITY;
            const int r = r0 + tid / w;
            float M = -INFINITY, L = 0.0f;
            if (r < R) {
                for (int s = tid % w; s < a.nsplit; s += 4 * w) {
                    v2f x[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = s + i * w < a.nsplit ? st[(int64_t)(s + i * w) * R + r] : v2f{-INFINITY, 0.0f};
                    const float mn = fmaxf(fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x)), M), mz = mn == -INFINITY ? 0.0f : mn;
                    L *= __builtin_amdgcn_exp2f(M - mz);
#pragma unroll
                    for (int i = 0; i < 4; i++) L = __builtin_fmaf(x[i].y, __builtin_amdgcn_exp2f(x[i].x - mz), L);
                    M = mn;
                }
            }
            for (int o = 1; o < w; o <<= 1) {
                const float mo = __shfl_xor(M, o, 64), lo = __shfl_xor(L, o, 64);
                const float mn = fmaxf(M, mo), mz = mn == -INFINITY ? 0.0f : mn;
                L = L * __builtin_amdgcn_exp2f(M - mz) + lo * __builtin_amdgcn_exp2f(mo - mz);
                M = mn;
            }
            __syncthreads();
            if (tid % w == 0) { sm[tid / w] = M == -INFINITY ? 0.0f : M; sl[tid / w] = L == 0.0f ? 0.0f : 1.0f / L; }
            __syncthreads();
            const int n = R - r0 < rows ? R - r0 : rows;
#pragma unroll
            for (int i = 0; i < 4; i++) if (i < n && s4[i] != -INFINITY) t = __builtin_fmaf(__builtin_amdgcn_exp2f(s4[i] - sm[i]), sl[i], t);
            for (int i0 = 4; i0 < n; i0 += 4) {
#pragma unroll
                for (int i = 0; i < 4; i++) s4[i] = j < a.n_kv && i0 + i < n ? lg[(int64_t)(r0 + i0 + i) * a.lpitch] : -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) if (i0 + i < n && s4[i] != -INFINITY) t = __builtin_fmaf(__builtin_amdgcn_exp2f(s4[i] - sm[i0 + i]), sl[i0 + i], t);
            }
        }
        if (j >= a.n_kv) return;
        if (a.mass_in) t += a.decay * ((const float *)(a.mass_in + hk * a.in_nb2 + i3 * a.in_nb3))[j];
        ((float *)(a.mass_out + hk * a.out_nb2 + i3 * a.out_nb3))[j] = t;
        return;
    }
    // a row of dst: D / 4 threads per slice of the sum over the splits
    constexpr int F4 = D / 4, SG = 256 / F4;
    __shared__ v4f so[SG][F4];
    const int r = blockIdx.x - mass_wgs, iq = m_query(a, r), h = hk * ratio + r - iq * ratio;
    const int f4 = tid % F4, sg = tid / F4;
    const bool in = 4 * f4 < a.dv;
    float M = -INFINITY;
    for (int s = tid; s < a.nsplit; s += 256) M = fmaxf(M, st[(int64_t)s * R + r].x);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((tid & 63) == 0) sm[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float ms = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = sg; s < a.nsplit; s += SG) {
        const v2f x = st[(int64_t)s * R + r];
        const v4f y = in ? *(const v4f *)(a.part + (base + (int64_t)s * R + r) * D + 4 * f4) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
        const float c = __builtin_amdgcn_exp2f(x.x - ms);
        L = __builtin_fmaf(x.y, c, L);
#pragma unroll
        for (int i = 0; i < 4; i++) O[i] = __builtin_fmaf(y[i], c, O[i]);
    }
    so[sg][f4] = O;
    if (f4 == 0) sl[sg] = L;
    __syncthreads();
    if (sg != 0 || !in) return;
#pragma unroll
    for (int i = 1; i < SG; i++) { O = O + so[i][f4]; L += sl[i]; }
    *(v4f *)((float *)(a.dst + (int64_t)h * a.d_nb1 + (int64_t)iq * a.d_nb2 + (int64_t)i3 * a.d_nb3) + 4 * f4) = L == 0.0f ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : O * (1.0f / L);
}

constexpr int STEP_WAVES = 4;

template <int TYPE, int D, bool HASV, int RP, bool RAW> static int step_launch(const MArgs & a, int ne3, hipStream_t s) {
    const int R = a.ratio * a.n_q;
    MI355_LAUNCH("fattn_mass_step", (mass_step_kernel<TYPE, D, STEP_WAVES, HASV, 1, RP, RAW>),
                 dim3((unsigned)(a.nsplit * ((R + 15) / 16)), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(STEP_WAVES * 64), 0, s, a);
    MI355_CHECK_LAUNCH();
    const int mass_wgs = (a.n_kv + 255) / 256;
    if (mass_wgs + (HASV ? R : 0) == 0) return MI355_OK;
    MI355_LAUNCH("fattn_mass_finish", mass_finish_kernel<D>, dim3((unsigned)(mass_wgs + (HASV ? R : 0)), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(256), 0, s, a, mass_wgs);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
static int step_d(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// rows of blocks that are whole pieces (see the kernel): full width, pieces aligned, a tile within 32-bit offsets
template <bool HASV> static bool step_raw(const MArgs & a) {
    const int D = step_d(a.d);
    uint64_t low = (uint64_t)(uintptr_t)a.k | a.k_nb1 | (uint64_t)a.k_nb2 | (uint64_t)a.k_nb3;
    if (HASV) low |= (uint64_t)(uintptr_t)a.v | a.v_nb1 | (uint64_t)a.v_nb2 | (uint64_t)a.v_nb3;
    return a.d == D && (!HASV || a.dv == D) && (low & (uint64_t)(D / 16 - 1)) == 0 && a.k_nb1 < (1u << 26) && (!HASV || a.v_nb1 < (1u << 26));
}
template <int TYPE, int D, bool HASV, bool RAW> static int step_rows(const MArgs & a, int ne3, hipStream_t s) {
    const int R = a.ratio * a.n_q;
    if constexpr (Fmt<TYPE>::quant && HASV && D <= 128) {
        if constexpr (D == 128) if (R <= 4) return step_launch<TYPE, D, HASV, 4, RAW>(a, ne3, s);
        if (R <= 8) return step_launch<TYPE, D, HASV, 8, RAW>(a, ne3, s);
    }
    return step_launch<TYPE, D, HASV, 16, RAW>(a, ne3, s);
}
template <int TYPE, bool HASV, bool RAW> static int step_size(const MArgs & a, int ne3, hipStream_t s) {
    switch (step_d(a.d)) {
        case 64:  return step_rows<TYPE, 64, HASV, RAW>(a, ne3, s);
        case 128: return step_rows<TYPE, 128, HASV, RAW>(a, ne3, s);
    }
    return step_rows<TYPE, 256, HASV, RAW>(a, ne3, s);
}
template <int TYPE, bool HASV> static int step_dispatch(const MArgs & a, int ne3, hipStream_t s) {
    if constexpr (Fmt<TYPE>::quant) if (step_raw<HASV>(a)) return step_size<TYPE, HASV, true>(a, ne3, s);
    return step_size<TYPE, HASV, false>(a, ne3, s);
}

// slices of the KV range: two workgroups per CU in all (what the registers allow), none with less than one 32-slot tile per wave
static int64_t step_splits(const mi355_fattn_args * p) {
    const int64_t R = p->n_head / p->n_head_kv * p->n_q, tiles = (p->n_kv + 31) / 32, base = p->n_head_kv * ((R + 15) / 16) * p->ne3;
    int64_t n = 512 / base, most = (tiles + STEP_WAVES - 1) / STEP_WAVES;
    if (n > most) n = most;
    if (n > 128) n = 128;
    return n < 1 ? 1 : n;
}

// ---- prompts ------------------------------------------------------------------------------------------------------------------------------
// one workgroup per (query, head, sequence): statistics
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
    const char * mrow = a.mask ? m_mask(a, iq, h, i3) : nullptr;
    const float slope = m_slope(a, h);
    const int64_t row = ((int64_t)i3 * a.n_head + h) * a.n_q + iq;
    float m = -INFINITY, l = 0.0f;
    for (int j = tid; j < a.n_kv; j += MT) {
        const float s = logit<TYPE>(a, q, kb + (int64_t)j * a.k_nb1, mrow, slope, j);
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
            __syncthreads();
            if (tid < a.d) q[tid] = ((const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3))[tid];
            __syncthreads();
            const char * mrow = a.mask ? m_mask(a, iq, h, i3) : nullptr;
            if (j < a.n_kv) s = logit<TYPE>(a, q, krow, mrow, m_slope(a, h), j);
            if (s != -INFINITY) t += expf(s - a.stats[row * 2]) * a.stats[row * 2 + 1];
        }
    if (j >= a.n_kv) return;
    if (a.mass_in) t += a.decay * ((const float *)(a.mass_in + hk * a.in_nb2 + i3 * a.in_nb3))[j];
    ((float *)(a.mass_out + hk * a.out_nb2 + i3 * a.out_nb3))[j] = t;
}

template <int TYPE> static int mass_launch(const MArgs & a, int ne3, hipStream_t s) {
    if (a.n_kv == 0) return MI355_OK;
    MI355_LAUNCH("fattn_mass_rows", mass_rows_kernel<TYPE>, dim3((unsigned)a.n_head, (unsigned)a.n_q, (unsigned)ne3), dim3(MT), 0, s, a);
    MI355_CHECK_LAUNCH();
    MI355_LAUNCH("fattn_mass", mass_slots_kernel<TYPE>, dim3((unsigned)((a.n_kv + MT - 1) / MT), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(MT), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}

// steps: [statistics][partial rows of dst][logits]; prompts: statistics
struct WsParts { int64_t nsplit, lpitch, stats, part, logits; };
static WsParts mass_parts(const mi355_fattn_args * p, bool with_dst) {
    const int64_t rows = p->ne3 * p->n_head * p->n_q;
    WsParts w = {1, 0, rows * 2, 0, 0};
    if (p->n_q <= MI355_MASS_MAX_Q) {
        w.nsplit = step_splits(p);
        w.lpitch = (p->n_kv + 3) / 4 * 4;
        w.stats = (w.nsplit * rows * 2 + 3) / 4 * 4;
        w.part = with_dst ? w.nsplit * rows * step_d(p->d) : 0;
        w.logits = rows * w.lpitch;
    }
    return w;
}
static int64_t mass_workspace(const mi355_fattn_args * p, bool with_dst) {
    if (!p || p->n_q < 0 || p->n_kv < 0 || p->n_head < 1 || p->n_head_kv < 1 || p->n_head % p->n_head_kv || p->ne3 < 1 || p->d < 8 || p->d > 256) return -1;
    const WsParts w = mass_parts(p, with_dst);
    return (w.stats + w.part + w.logits) * 4;
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
    if (p->mask && (p->m_ne2 < 1 || p->m_ne3 < 1 || p->m_ne2 > 0x7fffffff || p->m_ne3 > 0x7fffffff)) return MI355_E_SHAPE;
    if (p->k_nb1 < 0 || p->k_nb1 > 0x7fffffff || (with_dst && (p->v_nb1 < 0 || p->v_nb1 > 0x7fffffff))) return MI355_E_SHAPE;
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
    a.k = (const char *)p->k; a.k_nb1 = (uint32_t)p->k_nb1; a.k_nb2 = p->k_nb2; a.k_nb3 = p->k_nb3;
    a.v = (const char *)p->v; a.v_nb1 = (uint32_t)p->v_nb1; a.v_nb2 = p->v_nb2; a.v_nb3 = p->v_nb3;
    a.mask = (const char *)p->mask; a.m_nb1 = p->m_nb1; a.m_nb2 = p->m_nb2; a.m_nb3 = p->m_nb3; a.m_ne2 = (int)p->m_ne2; a.m_ne3 = (int)p->m_ne3;
    a.ratio = (int)(p->n_head / p->n_head_kv); a.by_ratio = a.ratio > 1 ? (uint32_t)(((1ull << 32) + a.ratio - 1) / a.ratio) : 0;
    a.dst = with_dst ? (char *)p->dst : nullptr; a.d_nb1 = p->d_nb1; a.d_nb2 = p->d_nb2; a.d_nb3 = p->d_nb3;
    a.mass_in = w->decay != 0.0f ? (const char *)w->mass_in : nullptr; a.in_nb2 = w->in_nb2; a.in_nb3 = w->in_nb3;
    a.mass_out = (char *)w->mass_out; a.out_nb2 = w->out_nb2; a.out_nb3 = w->out_nb3;
    a.n_q = (int)p->n_q; a.n_kv = (int)p->n_kv; a.n_head = (int)p->n_head; a.n_head_kv = (int)p->n_head_kv; a.d = (int)p->d; a.dv = (int)dv;
    a.scale = p->scale; a.max_bias = p->max_bias; a.logit_softcap = p->logit_softcap; a.decay = w->decay;
    a.n_head_log2 = 1u << (uint32_t)floorf(log2f((float)p->n_head));
    a.m0 = powf(2.0f, -(p->max_bias) / a.n_head_log2);
    a.m1 = powf(2.0f, -(p->max_bias / 2.0f) / a.n_head_log2);
    const WsParts parts = mass_parts(p, with_dst);
    a.nsplit = (int)parts.nsplit; a.lpitch = (int)parts.lpitch;
    a.stats = (float *)workspace;
    a.part = a.stats + parts.stats;
    a.logits = a.part + parts.part;
    hipStream_t s = (hipStream_t)stream;
    if (p->n_q <= MI355_MASS_MAX_Q) switch (p->type_k) {
        case MI355_TYPE_F16:  return with_dst ? step_dispatch<MI355_TYPE_F16, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_F16, false>(a, (int)p->ne3, s);
        case MI355_TYPE_BF16: return with_dst ? step_dispatch<MI355_TYPE_BF16, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_BF16, false>(a, (int)p->ne3, s);
        case MI355_TYPE_Q8_0: return with_dst ? step_dispatch<MI355_TYPE_Q8_0, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_Q8_0, false>(a, (int)p->ne3, s);
        case MI355_TYPE_Q4_0: return with_dst ? step_dispatch<MI355_TYPE_Q4_0, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_Q4_0, false>(a, (int)p->ne3, s);
    }
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
