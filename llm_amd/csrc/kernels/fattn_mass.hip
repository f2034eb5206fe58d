// fattn_mass.hip -- attention weight per cached slot: mi355_flash_attn_ext_mass (a decode step's attention together with it) and
// mi355_attn_mass (the weight alone, for a prompt's queries).
//
//   s_ij = scale q_i . k_j [softcap] + slope mask_ij      p_ij = exp(s_ij - m_i) / l_i     (m_i, l_i: maximum and sum over the slots i sees)
//   dst_i = sum_j p_ij v_j      mass_out[hk][j] = decay mass_in[hk][j] + sum over the heads of hk and all queries i of p_ij
// A slot that a query does not see (mask -inf) takes no part whatever its row holds, NaN included; a query that sees nothing gives a zero row and
// no weight.  Sums, maxima and logits are f32; what meets the matrix cores is 22 bits of q and p (two f16 parts), 24 over bf16 caches (three bf16
// parts), and the cache's own values, exact.
#include "common.h"
#include "spans.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct RowC { float qe, slope, m, inv; };      // per row: power of two of q, ALiBi slope (log2 domain), maximum, 1 / sum

struct MArgs {
    const char * q; int64_t q_nb1, q_nb2, q_nb3;
    const char * k; uint32_t k_nb1; int64_t k_nb2, k_nb3;        // (rows at most 2 GiB apart: a row's address is one 32 x 32 + 64 bit multiply-add)
    const char * v; uint32_t v_nb1; int64_t v_nb2, v_nb3;
    const char * mask; int64_t m_nb1, m_nb2, m_nb3; int m_ne2, m_ne3;
    char * dst; int64_t d_nb1, d_nb2, d_nb3;
    const char * mass_in; int64_t in_nb2, in_nb3;
    char * mass_out; int64_t out_nb2, out_nb3;
    int n_q, n_kv, n_head_kv, d, dv;
    float scale, max_bias, logit_softcap, m0, m1, decay;
    uint32_t n_head_log2;
    int ratio; uint32_t by_ratio;   // heads per KV head; ceil(2^32 / ratio), 0 for ratio 1 (r / ratio without a division)
    int nsplit, nchunk, lpitch, one;
    float * logits;     // steps: [ne3][n_head_kv][rows][lpitch], log2 domain
    float * stats;      // [ne3][n_head_kv][nsplit][rows][2]: maximum (log2 domain) and sum of a slice
    float * part;       // steps: [ne3][n_head_kv][nsplit][rows][D]; prompts: [ne3][n_head_kv][nchunk][n_kv]
    RowC * rowc;        // prompts: [ne3][n_head_kv][rows]
    uint8_t * cls; int cpitch;      // prompts: [m_ne3][m_ne2][n_q][cpitch] classes of the mask's 32-slot tiles
    uint16_t * qparts;  // prompts: [ne3][n_head_kv][rows][parts][D]
};

// value e of a row of f16 or bf16
template <int TYPE> static __device__ __forceinline__ float kv_value(const char * row, int e) {
    const uint16_t y = ((const uint16_t *)row)[e];
    return TYPE == MI355_TYPE_F16 ? h2f(y) : __uint_as_float((uint32_t)y << 16);
}

// row r of a KV head = (query, head of the group); r * ratio < 2^32
static __device__ __forceinline__ int m_query(const MArgs & a, int r) { return a.by_ratio ? (int)__umulhi((uint32_t)r, a.by_ratio) : r; }
static __device__ __forceinline__ const char * m_mask(const MArgs & a, int iq, int h, int i3) {
    return a.mask + iq * a.m_nb1 + (a.m_ne2 > 1 ? h % a.m_ne2 : 0) * a.m_nb2 + (a.m_ne3 > 1 ? i3 % a.m_ne3 : 0) * a.m_nb3;
}
// mass_out of a slot whose weight is t
static __device__ __forceinline__ void mass_store(const MArgs & a, int hk, int i3, int j, float t) {
    if (a.mass_in) t += a.decay * ((const float *)(a.mass_in + hk * a.in_nb2 + i3 * a.in_nb3))[j];
    ((float *)(a.mass_out + hk * a.out_nb2 + i3 * a.out_nb3))[j] = t;
}
// x[i] -> cap log2(e) tanh(x[i]), c2 = cap log2(e), off by a few 2^-24 of the result itself.  Below 5/8 it is x + x^3 P(x^2), P the least-maximum fit
// of (tanh x - x) / x^3 with 5 terms (relative error 2^-27.8); from there on 1 - 2 / (e^2|x| + 1), which would cancel nearer to 0 (2^-23 of the cap,
// however small the logit).  Logits seldom reach 5/8 of the cap, and a wave that has none there leaves the second form out: 2047 x 2047 bf16
// with a cap of 30 takes 221 us, with both forms at every logit 261 (or a cap of 3: 286), without a cap 157
template <int N> static __device__ __forceinline__ void cap_logits(float (&x)[N], float c2) {
    auto near = [](float x) {
        const float z = x * x;
        float p = __builtin_fmaf(z, -0.005717036779969931f, 0.020650578662753105f);
        p = __builtin_fmaf(z, p, -0.05374349653720856f);
        p = __builtin_fmaf(z, p, 0.13331490755081177f);
        p = __builtin_fmaf(z, p, -0.3333328366279602f);
        return __builtin_fmaf(x * z, p, x);
    };
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]));
    if (__any(top >= 0.625f)) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.0f * LOG2E * fabsf(x[i])) + 1.0f), 1.0f);
            x[i] = c2 * (fabsf(x[i]) < 0.625f ? near(x[i]) : copysignf(far, x[i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = c2 * near(x[i]);
    }
}
// exponent that brings a row's largest value to [2^14, 2^15)
static __device__ __forceinline__ int row_exp(float amax) { return amax > 0.0f && amax < INFINITY ? __builtin_amdgcn_frexp_expf(amax) - 15 : 0; }
static __device__ __forceinline__ float m_slope(const MArgs & a, uint32_t h) {
    if (!(a.max_bias > 0.0f)) return 1.0f;
    return h < a.n_head_log2 ? powf(a.m0, h + 1) : powf(a.m1, 2 * (h - a.n_head_log2) + 1);
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

// q and K in parts, sum over the parts p of q_p K: an infinity of K meets the parts' different signs and gives a NaN where the product is an infinity.
// Only the largest part, which has q's sign, meets it: the others take K without its non-finite values.  (Where q's large part is 0 so is q, next to
// its row's largest value.)  Nor does what is read in place of the features past the head size, which meets zeros of q.  For tiles that have a
// NaN among their products
template <bool BF> static __device__ __forceinline__ v4i finite(v4i x) { sanitize<BF>(x); return x; }
static __device__ __forceinline__ float max_or_nan(float x, float y) { return __builtin_elementwise_maximum(x, y); }

static __device__ __forceinline__ float max_groups(float v) {       // over the four 16-lane groups, lanes of equal place
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
static __device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// RP (blocks only): the 16 columns of a tile are RP rows times 16 / RP classes of 32-blocks -- at GQA 4 or 8
// the columns that would repeat a row each scale P by the blocks of their class, so a lane forms D / 32 / (16 / RP) scaled copies of P and not
// D / 32; a feature tile takes its result from the columns of its block's class.
// RAW (blocks only, step_raw): rows come in as consecutive pieces of D / 16 bytes (17 or 9 a row) and are taken apart in LDS, where otherwise a lane
// loads the 8 bytes of its own chunk at every second byte address.  Taken where it pays, raw_pays below.
// ONE: a workgroup has all slots of its KV head and finishes by itself, without the second launch (step_one).
template <int TYPE, int D, int NW, bool HASV, int RP, bool RAW, bool ONE>
__global__ void __launch_bounds__(NW * 64, D <= 64 && !ONE ? 3 : D <= 128 ? 2 : 1)
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
    __shared__ v4i qs[KS][P][64];
    uint8_t (&raw)[NW][VB] = lds;                               // RAW: raw rows of K, then of V, then V's values, one after the other
    static_assert(!RAW || VB >= 32 * PR * PB + 16, "raw rows fit");
    __shared__ __attribute__((aligned(16))) uint16_t kd[F::quant ? NW : 1][F::quant ? 32 * KS : 8], vd[F::quant && HASV ? NW : 1][F::quant && HASV ? 32 * KS : 8];
    __shared__ float wm[NW][16], wl[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const int ratio = a.ratio, R = ratio * a.n_q;
    const int hk = blockIdx.y, rb = blockIdx.x / a.nsplit * 16, i3 = blockIdx.z, split = blockIdx.x % a.nsplit;
    const char * kb = a.k + hk * a.k_nb2 + i3 * a.k_nb3;
    const char * vb = HASV ? a.v + hk * a.v_nb2 + i3 * a.v_nb3 : nullptr;
    const bool m8 = a.mask && (((uintptr_t)a.mask | (uintptr_t)a.m_nb1 | (uintptr_t)a.m_nb2 | (uintptr_t)a.m_nb3) & 7) == 0;
    const bool capped = a.logit_softcap != 0.0f;
    // this lane's row (columns past the last one repeat it)
    const int r = rb + lr % RP < R ? rb + lr % RP : R - 1, iq = m_query(a, r), h = hk * ratio + r - iq * ratio;
    const char * mrow = m_mask(a, iq, h, i3);

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
    auto load_mask = [&](int t, u2 (&w)[2]) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int j = 32 * t + 16 * u + 4 * g;
            if (m8 && j + 4 <= a.n_kv) w[u] = *(const u2 *)(mrow + 2 * (int64_t)j);
            else {
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = j + i >= a.n_kv ? 0xfc00u : a.mask ? ((const uint16_t *)mrow)[j + i] : 0u;
                w[u] = u2{y[0] | y[1] << 16, y[2] | y[3] << 16};
            }
        }
    };
    auto sees = [&](const u2 (&w)[2]) { return __any(!(w[0].x == 0xfc00fc00u && w[0].y == 0xfc00fc00u && w[1].x == 0xfc00fc00u && w[1].y == 0xfc00fc00u)); };

    // tiles are dealt to the waves of all slices in turn: sequences shorter than the range keep them all busy.  A tile hidden from every row
    // costs its mask, which runs one tile ahead of the rows; the first tile is fetched without asking: one round trip instead of two
    int t = split * NW + wave;
    u2 mk[2], mkn[2];
    if (t < ntiles) { load_k(t); load_v(t); load_mask(t, mk); }
    if (t + TW < ntiles) load_mask(t + TW, mkn);

    // q for all waves, in LDS as the B operand takes it: a wave splits the 32-feature chunks that fall to it.  Scale and log2(e) go on q; for f16
    // the row's largest value is brought to [2^14, 2^15) by a power of two that the logits get back (its small values then stay clear of the
    // subnormal range)
    constexpr int QN = (KS + NW - 1) / NW;
    float y[QN][8], amax = 0.0f;
    const float slope = m_slope(a, h) * LOG2E, sc = capped ? a.scale / a.logit_softcap : a.scale * LOG2E;
    const float * qp = (const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3);
#pragma unroll
    for (int n = 0; n < QN; n++) {
        const int f = 32 * (wave + NW * n) + 8 * g;
        v4f y0 = {0.0f, 0.0f, 0.0f, 0.0f}, y1 = y0;
        if (f < a.d) { y0 = *(const v4f *)(qp + f) * sc; y1 = *(const v4f *)(qp + f + 4) * sc; }
#pragma unroll
        for (int i = 0; i < 4; i++) { y[n][i] = y0[i]; y[n][4 + i] = y1[i]; amax = fmaxf(amax, fmaxf(fabsf(y0[i]), fabsf(y1[i]))); }
    }
    int e = 0;
    if constexpr (!F::bf) {
        amax = max_groups(amax);
        if (g == 0) wm[wave][lr] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) amax = fmaxf(amax, wm[w][lr]);
        e = row_exp(amax);
    }
    const float qe = ldexpf(1.0f, e);
#pragma unroll
    for (int n = 0; n < QN; n++) {
        if (wave + NW * n >= KS) continue;
        v4i w[P];
#pragma unroll
        for (int i = 0; i < 8; i++) y[n][i] = ldexpf(y[n][i], -e);
        split8<F::bf, P>(y[n], w);
#pragma unroll
        for (int p = 0; p < P; p++) qs[wave + NW * n][p][lane] = w[p];
    }
    __syncthreads();

    float m = -INFINITY, l = 0.0f;      // of this lane's row; l over this lane's slots only
    int E = -64;                        // blocks: o holds 2^(14 - E) times its value, E the exponent of the largest scale of V met so far
    v4f o[HASV ? FT : 1];
#pragma unroll
    for (int i = 0; i < (HASV ? FT : 1); i++) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float * lg = a.logits + (((int64_t)i3 * a.n_head_kv + hk) * R + r) * a.lpitch;
    const bool mine = lr < RP && rb + lr < R;           // the lane that stores row r

    while (t < ntiles) {
        const u2 mc[2] = {mk[0], mk[1]};
        int tn = t + TW;                        // the next tile that a row sees
        while (tn < ntiles && !sees(mkn)) {
            if (mine) {
#pragma unroll
                for (int u = 0; u < 2; u++) if (32 * tn + 16 * u + 4 * g < a.lpitch) *(v4f *)(lg + 32 * tn + 16 * u + 4 * g) = v4f{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            }
            tn += TW;
            if (tn < ntiles) load_mask(tn, mkn);
        }
        const bool next = tn < ntiles;
        mk[0] = mkn[0]; mk[1] = mkn[1];
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
        v4f c[2];
        {
            hk_t dk[2][4];
            if constexpr (F::quant) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) dk[u][i] = *(const hk_t *)&kd[wave][(16 * u + 4 * g + i) * KS];
            }
            c[0] = c[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                v4i qv[P];
#pragma unroll
                for (int p = 0; p < P; p++) qv[p] = qs[ks][p][lane];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    v4i kop;
                    if constexpr (RAW) kop = raw_chunk<TYPE>(raw[wave] + (16 * u + lr) * PR * PB, 4 * ks + g).operand(g);
                    else if constexpr (F::quant) kop = *(const v4i *)(lds[wave] + (16 * u + lr) * VP + (4 * ks + g) * 16);
                    else kop = kc[u][ks].operand(g);
                    v4f b = F::quant ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : c[u];
#pragma unroll
                    for (int p = P - 1; p >= 0; p--) b = mfma16<F::bf>(kop, qv[p], b);
                    if constexpr (F::quant) {
#pragma unroll
                        for (int i = 0; i < 4; i++) c[u][i] = __builtin_fmaf(b[i], (float)dk[u][i][ks], c[u][i]);
                    } else c[u] = b;
                }
            }
            if constexpr (!F::quant) {                          // an infinity in a row of K (see finite)
                bool nan = false;
#pragma unroll
                for (int i = 0; i < 8; i++) nan |= c[i >> 2][i & 3] != c[i >> 2][i & 3];
                if (__builtin_expect(__any(nan), 0)) {
                    int again = lane;
                    asm("" : "+v"(again));                      // (q read again: what the products above read is not kept for this)
                    c[0] = c[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const v4i f = finite<F::bf>(kc[u][ks].raw), k0 = 4 * ks + g < a.d / 8 ? kc[u][ks].raw : f;
#pragma unroll
                            for (int p = P - 1; p >= 0; p--) c[u] = mfma16<F::bf>(p == 0 ? k0 : f, qs[ks][p][again], c[u]);
                        }
                }
            }
        }
        if (next) load_k(tn);                   // in flight during the rest of this tile
        if (tn + TW < ntiles) load_mask(tn + TW, mkn);
        float s[8], p[8];           // slots 32 t + 16 (i >> 2) + 4 g + (i & 3)
        bool some = false;                      // some row does not see some slot of the tile
        float mx = m;
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = c[i >> 2][i & 3] * qe;
        if (capped) cap_logits(s, a.logit_softcap * LOG2E);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float mv = h2f((uint16_t)(mc[i >> 2][(i & 3) >> 1] >> (16 * (i & 1))));
            s[i] = mv == -INFINITY ? -INFINITY : __builtin_fmaf(mv, slope, s[i]);
            mx = fmaxf(mx, s[i]);
            some |= s[i] == -INFINITY;
        }
        if (mine) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int j = 32 * t + 16 * u + 4 * g;
                if (j < a.lpitch) *(v4f *)(lg + j) = v4f{s[4 * u], s[4 * u + 1], s[4 * u + 2], s[4 * u + 3]};
            }
        }
        mx = max_groups(mx);
        const float ms = mx == -INFINITY ? 0.0f : mx;
        float corr = __builtin_amdgcn_exp2f(m - ms);        // m = -inf: 0
        l *= corr;
#pragma unroll
        for (int i = 0; i < 8; i++) { p[i] = __builtin_amdgcn_exp2f(s[i] - ms); l += p[i]; }
        m = mx;
        if constexpr (HASV) {
            const bool hidden = __any(some);
            _Float16 dd[SETS][8];
            if constexpr (RAW) { put_raw(vp); raw_scales(vd[wave]); __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
            if constexpr (F::quant) {
                // the scales of V go on P, those of this lane's class of blocks.  A hidden slot's is taken as 0 (it may be NaN)
                _Float16 dm = 0;
#pragma unroll
                for (int q = 0; q < SETS; q++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int b = q * NC + lr / RP;
                        dd[q][i] = __builtin_bit_cast(_Float16, vd[wave][(16 * (i >> 2) + 4 * g + (i & 3)) * KS + (b < KS ? b : 0)]);
                    }
                if (hidden) {
#pragma unroll
                    for (int q = 0; q < SETS; q++)
#pragma unroll
                        for (int i = 0; i < 8; i++) if (s[i] == -INFINITY) dd[q][i] = 0;
                }
#pragma unroll
                for (int q = 0; q < SETS; q++)
#pragma unroll
                    for (int i = 0; i < 8; i++) dm = __builtin_elementwise_max(dm, __builtin_elementwise_abs(dd[q][i]));
                const float dmx = max_groups((float)dm);
                const int e = dmx > 0.0f && dmx < INFINITY ? __builtin_amdgcn_frexp_expf(dmx) - 1 : -64;
                const int En = E > e ? E : e;
                corr = ldexpf(corr, E - En);
                E = En;
            }
            if (__any(corr != 1.0f)) {
#pragma unroll
                for (int i = 0; i < FT; i++) o[i] = o[i] * corr;
            }
            // ---- V tile into LDS.  A slot that some row does not see must not reach that row through 0 * NaN: its non-finite values are
            // taken out here and added below to the rows that do see it
            uint32_t bad = 0;                                   // slots of the tile with values taken out
            if constexpr (!F::quant) if (hidden) {
                uint32_t unseen = 0;                            // bit j: slot 32 t + j is hidden from some row
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint64_t b = __ballot(s[i] == -INFINITY);
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
            v4i pf[P];
            if constexpr (!F::bf) {                             // f16 parts: clear of the subnormal range
                const float up = F::quant ? ldexpf(1.0f, 14 - E) : 16384.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] *= up;
            }
            if constexpr (!F::quant) split8<F::bf, P>(p, pf);
#pragma unroll
            for (int f = 0; f < FT; f++) {
                if constexpr (F::quant) {
                    if (f % (FT / SETS) == 0) {                 // the next scaled copy
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) y[i] = p[i] * (float)dd[f / (FT / SETS)][i];
                        split8<false, 2>(y, pf);
                    }
                }
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(vt + 32 * f));
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(vt + 32 * f + 16 * VP));
                v4i vop;
                __builtin_memcpy(&vop, &lo, 8);
                __builtin_memcpy((char *)&vop + 8, &hi, 8);
#pragma unroll
                for (int q = P - 1; q >= 0; q--) o[f] = mfma16<F::bf>(vop, pf[q], o[f]);
            }
            if constexpr (!F::quant) if (bad) {                 // non-finite values of slots that only some rows see
                for (int row = 0; row < 32; row++) {
                    if (!(bad >> row & 1)) continue;
                    const int from = ((row & 15) >> 2) * 16 + lr, i = (row >> 4) * 4 + (row & 3), j = 32 * t + row;
                    if (j >= a.n_kv) continue;
                    const char * vr = vb + (uint64_t)(uint32_t)j * a.v_nb1;
                    float pr = 0.0f, sr = -INFINITY;
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        const float a0 = __shfl(p[q], from, 64), a1 = __shfl(s[q], from, 64);
                        if (q == i) { pr = a0; sr = a1; }
                    }
#pragma unroll
                    for (int f = 0; f < FT; f++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int e = 16 * f + 4 * g + q;
                            if (e >= a.dv) continue;
                            const float y = kv_value<TYPE>(vr, e);
                            if (sr != -INFINITY && !(fabsf(y) < INFINITY)) o[f][q] += pr * y;
                        }
                }
            }
        }
        t = tn;
    }
    // ---- the waves' states meet in LDS
    l = sum_groups(l);
    if (g == 0 && lr < RP) { wm[wave][lr] = m; wl[wave][lr] = l; }
    if constexpr (HASV) {
        float * ob = (float *)lds[wave] + lr % RP * OP + 4 * g;
        const float back = F::bf ? 1.0f : F::quant ? ldexpf(1.0f, E - 14) : 1.0f / 16384.0f;
#pragma unroll
        for (int f = 0; f < FT; f++) if (NC == 1 || f / 2 % NC == lr / RP) *(v4f *)(ob + 16 * f) = o[f] * back;
    }
    __syncthreads();
    const int rows = R - rb < RP ? R - rb : RP;
    if constexpr (ONE) {
        __shared__ float rm[16], ri[16];
        if (tid < rows) {
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][tid]);
            const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < NW; w++) L = __builtin_fmaf(wl[w][tid], __builtin_amdgcn_exp2f(wm[w][tid] - ms), L);
            rm[tid] = ms; ri[tid] = L == 0.0f ? 0.0f : 1.0f / L;
        }
        __threadfence_block();                                  // (the logits of all waves, read below)
        __syncthreads();
        const float * all = a.logits + ((int64_t)i3 * a.n_head_kv + hk) * R * a.lpitch;
        for (int j = tid; j < a.n_kv; j += NW * 64) {
            float x[16], w = 0.0f;
#pragma unroll
            for (int rr = 0; rr < 16; rr++) x[rr] = rr < rows ? all[(int64_t)rr * a.lpitch + j] : -INFINITY;
#pragma unroll
            for (int rr = 0; rr < 16; rr++) if (x[rr] != -INFINITY) w = __builtin_fmaf(__builtin_amdgcn_exp2f(x[rr] - rm[rr]), ri[rr], w);
            mass_store(a, hk, i3, j, w);
        }
        if constexpr (HASV) {
            for (int idx = tid; idx < rows * (D / 4); idx += NW * 64) {
                const int rr = idx / (D / 4), f4 = idx % (D / 4), q = m_query(a, rr), hr = hk * ratio + rr - q * ratio;
                if (4 * f4 >= a.dv) continue;
                v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < NW; w++) O = O + *(const v4f *)((const float *)lds[w] + rr * OP + 4 * f4) * __builtin_amdgcn_exp2f(wm[w][rr] - rm[rr]);
                *(v4f *)((float *)(a.dst + (int64_t)hr * a.d_nb1 + (int64_t)q * a.d_nb2 + (int64_t)i3 * a.d_nb3) + 4 * f4) = ri[rr] == 0.0f ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : O * ri[rr];
            }
        }
        return;
    }
    const int64_t base = (((int64_t)i3 * a.n_head_kv + hk) * a.nsplit + split) * R + rb;
    if constexpr (HASV) {
        for (int idx = tid; idx < rows * (D / 4); idx += NW * 64) {
            const int rr = idx / (D / 4), f4 = idx % (D / 4);
            if (4 * f4 >= a.dv) continue;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][rr]);
            const float ms = M == -INFINITY ? 0.0f : M;
            v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < NW; w++) O = O + *(const v4f *)((const float *)lds[w] + rr * OP + 4 * f4) * __builtin_amdgcn_exp2f(wm[w][rr] - ms);
            *(v4f *)(a.part + (base + rr) * D + 4 * f4) = O;
        }
    }
    if (tid < rows) {
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][tid]);
        const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < NW; w++) L = __builtin_fmaf(wl[w][tid], __builtin_amdgcn_exp2f(wm[w][tid] - ms), L);
        *(v2f *)(a.stats + (base + tid) * 2) = v2f{M, L};
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
        if (j < a.n_kv) mass_store(a, hk, i3, j, t);
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
constexpr int one_waves(int D) { return D <= 128 ? 8 : 4; }     // what the LDS holds

template <int TYPE, int D, bool HASV, int RP, bool RAW> static int step_launch(const MArgs & a, int ne3, hipStream_t s) {
    const int R = a.ratio * a.n_q;
    MI355_LAUNCH("fattn_mass_step", (mass_step_kernel<TYPE, D, STEP_WAVES, HASV, RP, RAW, false>),
                 dim3((unsigned)(a.nsplit * ((R + 15) / 16)), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(STEP_WAVES * 64), 0, s, a);
    MI355_CHECK_LAUNCH();
    const int mass_wgs = (a.n_kv + 255) / 256;
    if (mass_wgs + (HASV ? R : 0) == 0) return MI355_OK;
    MI355_LAUNCH("fattn_mass_finish", mass_finish_kernel<D>, dim3((unsigned)(mass_wgs + (HASV ? R : 0)), (unsigned)a.n_head_kv, (unsigned)ne3), dim3(256), 0, s, a, mass_wgs);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
static int step_d(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Are rows of blocks taken in as pieces (see the kernel)?  Whole call, 8 KV heads, own chunks against pieces, us.  Pieces hold more registers, at D 64
// and for q8_0 with V more than there are beside two or three waves:
//   q8_0 with V  D 64: 6 x 32768, 4 / 20 rows  80 / 156 against 108 / 259;  D 128: the same 112 / 201 against 112 / 252, 8 x 4099, 4 / 12 rows
//                30.6 / 35.0 against 32.1 / 39.7;  D 256: 4 x 32768, 4 rows  162 against 165, 8 x 4099, 4 / 20 rows  68 / 113 against 67 / 111
//   q4_0 with V  D 64: 6 x 32768, 4 / 20 rows  70 / 152 against 72 / 156;  D 128: 102 / 198 against 99 / 198;  D 256: 4 x 32768  159 against 150
//   without V    6 x 32768, 32 rows  D 64 q8_0 148 against 147, q4_0 146 against 144;  D 128 q8_0 181 against 169, q4_0 180 against 159
template <int TYPE, int D, bool HASV> constexpr bool raw_pays() { return Fmt<TYPE>::quant && D > 64 && !(TYPE == MI355_TYPE_Q8_0 && D == 128 && HASV); }
// and can they be: full width, pieces aligned, a tile within 32-bit offsets
template <int D, bool HASV> static bool step_raw(const MArgs & a) {
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
template <int TYPE, int D, bool HASV> static int one_launch(const MArgs & a, int ne3, hipStream_t s) {
    MI355_LAUNCH("fattn_mass_one", (mass_step_kernel<TYPE, D, one_waves(D), HASV, 16, false, true>), dim3(1, (unsigned)a.n_head_kv, (unsigned)ne3), dim3(one_waves(D) * 64), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
template <int TYPE, int D, bool HASV> static int step_size(const MArgs & a, int ne3, hipStream_t s) {
    if (a.one) return one_launch<TYPE, D, HASV>(a, ne3, s);
    if constexpr (raw_pays<TYPE, D, HASV>()) if (step_raw<D, HASV>(a)) return step_rows<TYPE, D, HASV, true>(a, ne3, s);
    return step_rows<TYPE, D, HASV, false>(a, ne3, s);
}
template <int TYPE, bool HASV> static int step_dispatch(const MArgs & a, int ne3, hipStream_t s) {
    switch (step_d(a.d)) {
        case 64:  return step_size<TYPE, 64, HASV>(a, ne3, s);
        case 128: return step_size<TYPE, 128, HASV>(a, ne3, s);
    }
    return step_size<TYPE, 256, HASV>(a, ne3, s);
}

// One launch: a row tile of queries, and no more slots than one tile a wave.  8 heads of 128, f16, GPU time: 1 / 128 / 256 slots 8.4 / 7.8 / 9.5 us against
// 9.9 / 9.5 / 9.7 of the two launches (512 slots: 12.9 against 9.7), and 3 us less of the host's
static bool step_one(const mi355_fattn_args * p) {
    return p->n_head / p->n_head_kv * p->n_q <= 16 && p->n_kv <= 32 * one_waves(step_d(p->d));
}
// slices of the KV range: two workgroups per CU in all (what the registers allow), none with less than one 32-slot tile per wave
static int64_t step_splits(const mi355_fattn_args * p) {
    const int64_t R = p->n_head / p->n_head_kv * p->n_q, tiles = (p->n_kv + 31) / 32, base = p->n_head_kv * ((R + 15) / 16) * p->ne3;
    int64_t n = 512 / base, most = (tiles + STEP_WAVES - 1) / STEP_WAVES;
    if (n > most) n = most;
    if (n > 128) n = 128;
    return n < 1 ? 1 : n;
}

// ---- prompts: any number of queries, the weights alone ---------------------------------------------------------------------------------------
//
// Keeping the logits would move 8 bytes per (query, slot) pair; computing them twice costs 2 d products each on the matrix cores, which is less:
//   prompt_prep   q as two f16 (bf16 caches: three bf16) parts, scale and log2(e) on it, f16 rows brought to [2^14, 2^15) by a power of two; what
//                 each 32-slot tile of the mask is to each query
//   prompt_stats  S^T = K Q^T, a running maximum and sum per row: a wave holds 32 rows of Q in registers, K passes through LDS
//   prompt_mass   S^T again and sum over the rows of 2^(s - m) / l: a wave holds 32 or 64 slots of K, Q passes through LDS; the sums stay in
//                 registers, one per (slot, lane), and meet across the lanes once at the end
//   prompt_sum    the row chunks' sums and decay * mass_in, in a fixed order
// v_mfma_f32_32x32x16 throughout: K of f16 and bf16 as it is; blocks as their integers, whose products a block's scale is put on in f32.  On its way
// through LDS: K of f16 and bf16 in the first pass by DMA, two tiles ahead of the products, blocks through registers, one ahead; Q in the second pass
// by DMA, two tiles ahead, one with heads above 128 (LDS).  A tile that the mask hides from all rows of a wave (half of a causal prompt) costs its
// loads and its meeting.
// 64 queries x 32 heads over 16384 f16 slots: 6 + 24 + 5 + 32 us.  A pass is 17 GFLOP, 15 us at the rate a large product reaches here, behind 5 us
// until the first tile of 512 workgroups is there; without its products the first pass takes 20, without its exponentials 23.  2047
// causal queries, bf16: 16 + 69 + 79 + 5 us, 45 a pass at that rate.  Matrix cores and vector units are each busy a third of either pass (30-40 %), a
// wave waits for its turn or its operands most of the rest: 1.7 waves a SIMD do not cover one another's chains.
typedef float v16f __attribute__((ext_vector_type(16)));
constexpr int PT = 256;                  // threads: 4 waves
constexpr int PA_ROWS = 128, PA_SLOTS = 64, PB_ROWS = 32;

template <bool BF> static __device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else              return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// 64 lanes x 16 (4) bytes, each from its own address, to consecutive places in LDS.  Counted by vmcnt; the compiler does not know of them: it
// waits for too many loads where it waits for its own, never for too few
static __device__ __forceinline__ void dma16(const void * src, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory");
}
static __device__ __forceinline__ void dma4(const void * src, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory");
}
static __device__ __forceinline__ uint32_t lds_at(const void * p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}
// all but this wave's N newest loads and all its LDS reads are done, then the workgroup meets
template <int N> static __device__ __forceinline__ void wait_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// a value that was loaded, waited for here: a wait of the compiler's own in a loop that DMA runs through would wait for the DMA as well
static __device__ __forceinline__ void arrived(v4i & x) { asm volatile("" : "+v"(x)); }
static __device__ __forceinline__ void arrived(float & x) { asm volatile("" : "+v"(x)); }
// Rows of D 16-bit values in LDS, 16-byte chunks: chunk c of row r lies at c ^ (r & swz<D>()), so that a chunk's column is read without
// bank conflicts and a DMA's places stay consecutive
template <int D> constexpr int swz() { return D == 128 ? 15 : 7; }
template <int D> static __device__ __forceinline__ int lds_chunk(int r, int c) { return r * D * 2 + ((c ^ (r & swz<D>())) * 16); }

// What a 32-slot tile of the mask is to a query: nothing visible, all of it zero, or anything else (the tile past the last slot too).  Looked up
// by both passes and by every head that shares the mask, so that they read the mask itself only where it is neither (the diagonal of a prompt).
// No mask: one row of classes for all.  A row goes on to the end of the last workgroup's slots.
enum { MASK_HIDDEN = 0, MASK_ZERO = 1, MASK_MIXED = 2 };

// workgroups 0 .. class_wgs - 1: classes of 4 queries x 1024 slots.  The others: 16 rows of q -> parts, RowC; 16 lanes a row
template <int D, bool BF>
__global__ void __launch_bounds__(PT)
prompt_prep_kernel(const MArgs a, uint32_t class_wgs, uint32_t slot_wgs, uint32_t query_wgs, uint32_t row_wgs) {
    if (blockIdx.x < class_wgs) {
        const uint32_t y = blockIdx.x / slot_wgs, x = blockIdx.x - y * slot_wgs, plane = y / query_wgs;
        const int lane = threadIdx.x & 63, iq = (int)(y - plane * query_wgs) * 4 + (threadIdx.x >> 6);
        const int n_q = a.mask ? a.n_q : 1;
        if (iq >= n_q) return;
        const char * mrow = a.mask + iq * a.m_nb1 + plane % a.m_ne2 * a.m_nb2 + plane / a.m_ne2 * a.m_nb3;
        uint8_t * out = a.cls + ((int64_t)plane * n_q + iq) * a.cpitch;
        const int j0 = x * 1024;
        uint16_t v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) { const int j = j0 + 64 * i + lane; v[i] = j >= a.n_kv ? 0xfc00 : a.mask ? ((const uint16_t *)mrow)[j] : 0; }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int at = (j0 + 64 * i) / 32 + lane;
            const uint64_t hid = __ballot(v[i] == 0xfc00), zero = __ballot((v[i] & 0x7fff) == 0);
            if (lane < 2 && at < a.cpitch) {
                const uint32_t h = (uint32_t)(hid >> (32 * lane)), z = (uint32_t)(zero >> (32 * lane));
                out[at] = h == 0xffffffffu ? MASK_HIDDEN : z == 0xffffffffu ? MASK_ZERO : MASK_MIXED;
            }
        }
        return;
    }
    constexpr int NF = D / 128 > 0 ? D / 128 : 1, P = BF ? 3 : 2;   // chunks of 8 features per lane, parts
    const uint32_t w = blockIdx.x - class_wgs, y_ = w / row_wgs;
    const int lane = threadIdx.x & 15, hk = y_ % a.n_head_kv, i3 = y_ / a.n_head_kv, R = a.ratio * a.n_q;
    const int r = (int)(w - y_ * row_wgs) * (PT / 16) + (threadIdx.x >> 4);
    if (r >= R) return;
    const int iq = m_query(a, r), h = hk * a.ratio + r - iq * a.ratio;
    const float * qp = (const float *)(a.q + iq * a.q_nb1 + h * a.q_nb2 + i3 * a.q_nb3);
    const float sc = a.logit_softcap != 0.0f ? a.scale / a.logit_softcap : a.scale * LOG2E;
    float y[NF][8], amax = 0.0f;
#pragma unroll
    for (int n = 0; n < NF; n++) {
        const int f = 8 * (lane + 16 * n);
        v4f y0 = {0.0f, 0.0f, 0.0f, 0.0f}, y1 = y0;
        if (f < a.d) { y0 = *(const v4f *)(qp + f) * sc; y1 = *(const v4f *)(qp + f + 4) * sc; }
#pragma unroll
        for (int i = 0; i < 4; i++) { y[n][i] = y0[i]; y[n][4 + i] = y1[i]; amax = fmaxf(amax, fmaxf(fabsf(y0[i]), fabsf(y1[i]))); }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    const int e = BF ? 0 : row_exp(amax);
    const int64_t row = ((int64_t)i3 * a.n_head_kv + hk) * R + r;
#pragma unroll
    for (int n = 0; n < NF; n++) {
        if (lane + 16 * n >= D / 8) continue;
        v4i part[P];
#pragma unroll
        for (int i = 0; i < 8; i++) y[n][i] = ldexpf(y[n][i], -e);
        split8<BF, P>(y[n], part);
#pragma unroll
        for (int p = 0; p < P; p++) *(v4i *)(a.qparts + (row * P + p) * D + 8 * (lane + 16 * n)) = part[p];
    }
    if (lane == 0) { a.rowc[row].qe = ldexpf(1.0f, e); a.rowc[row].slope = m_slope(a, h) * LOG2E; }
}

// blocks: the products of a 32-block's integers take their slots' scales (of the 16 slots that this lane's accumulator holds) and join the sums
static __device__ __forceinline__ void fold_block(const uint16_t * scales, int lh, const v16f & part, v16f & c) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const h4 d = *(const h4 *)(scales + 8 * q + 4 * lh);
#pragma unroll
        for (int i = 0; i < 4; i++) c[4 * q + i] = __builtin_fmaf(part[4 * q + i], (float)d[i], c[4 * q + i]);
    }
    asm volatile("" : "+v"(c));                                 // (put off, the sums of all blocks would have to be held: they do not fit)
}

// logits (log2 domain) of a 32 x 32 tile from slot j0 on, in place of its products: sc what they lack, cl the tile's class for this lane's query
template <bool CAP> static __device__ __forceinline__ void tile_logits(const MArgs & a, v16f & c, float sc, float slope, int cl, const char * mrow, bool m8, int j0) {
#pragma unroll
    for (int i = 0; i < 16; i++) c[i] *= sc;
    if constexpr (CAP) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = c[i];
        cap_logits(x, a.logit_softcap * LOG2E);
#pragma unroll
        for (int i = 0; i < 16; i++) c[i] = x[i];
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {                               // slot 8 q + 4 (lane / 32) + i
        const int j = j0 + 8 * q + 4 * ((threadIdx.x >> 5) & 1);
        u2 w;
        if (cl != MASK_MIXED) w = u2{0u, 0u};
        else if (m8 && j + 4 <= a.n_kv) w = *(const u2 *)(mrow + 2 * (int64_t)j);
        else {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = j + i >= a.n_kv ? 0xfc00u : a.mask ? ((const uint16_t *)mrow)[j + i] : 0u;
            w = u2{y[0] | y[1] << 16, y[2] | y[3] << 16};
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float mv = cl == MASK_HIDDEN ? -INFINITY : h2f((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
            c[4 * q + i] = mv == -INFINITY ? -INFINITY : __builtin_fmaf(mv, slope, c[4 * q + i]);
        }
    }
}
static __device__ __forceinline__ const uint8_t * class_row(const MArgs & a, int iq, int h, int i3) {
    if (!a.mask) return a.cls;
    const int plane = (a.m_ne3 > 1 ? i3 % a.m_ne3 : 0) * a.m_ne2 + (a.m_ne2 > 1 ? h % a.m_ne2 : 0);
    return a.cls + ((int64_t)plane * a.n_q + iq) * a.cpitch;
}

// statistics of a row -> maximum (0: sees nothing) and 1 / sum
static __device__ __forceinline__ v2f row_result(float M, float L) { return v2f{M == -INFINITY ? 0.0f : M, L == 0.0f ? 0.0f : 1.0f / L}; }
// Workgroups come to the CUs in turn, so a CU holds those a multiple of 256 apart: under a causal mask the same place of another head, twice the
// longest on one CU and twice the shortest on another.  Heads of every second 256 workgroups take their places from the other end
// (2047 x 2047: 82 + 95 -> 67 + 87 us)
static __device__ __forceinline__ bool turned() { return (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x / 256 & 1; }

template <int TYPE, int D, bool CAP>
__global__ void __launch_bounds__(PT, D <= 128 ? 2 : 1)
prompt_stats_kernel(const MArgs a) {
    typedef Fmt<TYPE> F;
    constexpr int KS = D / 16, QP = F::parts, S = F::quant ? 2 : 3;      // S: tiles in LDS
    constexpr int RS = PT / (D / 8), CN = PA_SLOTS / RS;        // rows a pass of the workgroup's chunks covers, passes of a tile
    __shared__ __attribute__((aligned(16))) uint8_t kt[S][PA_SLOTS * D * 2];
    __shared__ __attribute__((aligned(16))) uint16_t kd[F::quant ? S : 1][F::quant ? D / 32 : 1][PA_SLOTS];
    __shared__ uint32_t cl[S][PT / 64][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, lh = lane >> 5;
    const int R = a.ratio * a.n_q, hk = blockIdx.y, i3 = blockIdx.z, split = blockIdx.x % a.nsplit;      // the last rows first: a causal mask lets them see most
    const int rt = (int)(turned() ? blockIdx.x : gridDim.x - 1 - blockIdx.x) / a.nsplit * PA_ROWS, r_ = rt + wave * 32 + lr, r = r_ < R ? r_ : R - 1;
    const int iq = m_query(a, r), h = hk * a.ratio + r - iq * a.ratio;
    const char * kb = a.k + hk * a.k_nb2 + i3 * a.k_nb3;
    const char * mrow = m_mask(a, iq, h, i3);
    const uint8_t * crow = class_row(a, iq, h, i3);
    const bool m8 = a.mask && (((uintptr_t)a.mask | (uintptr_t)a.m_nb1 | (uintptr_t)a.m_nb2 | (uintptr_t)a.m_nb3) & 7) == 0;
    const bool mine = rt + wave * 32 < R;
    const int64_t row = ((int64_t)i3 * a.n_head_kv + hk) * R + r;
    const int nt = (a.n_kv + PA_SLOTS - 1) / PA_SLOTS, ns = a.nsplit;

    v4i qf[KS][QP];
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int p = 0; p < QP; p++) qf[ks][p] = *(const v4i *)(a.qparts + (row * QP + p) * D + 16 * ks + 8 * lh);
    float qe = a.rowc[row].qe, slope = a.rowc[row].slope;

    // this lane's chunk of a pass: chunks past the head size re-read the last one and meet zeros of q, slots past the end the last one and are hidden
    const int pos = tid % (D / 8), j_ = tid / (D / 8), c_ = F::quant ? pos : pos ^ (j_ & swz<D>()), cc = c_ < a.d / 8 ? c_ : a.d / 8 - 1;
    Chunk<F::quant ? TYPE : (int)MI355_TYPE_Q8_0> kr[F::quant ? CN : 1];
    uint16_t kdr[F::quant ? CN : 1];
    uint64_t off[CN];                                           // of this lane's chunks in a tile
#pragma unroll
    for (int i = 0; i < CN; i++) off[i] = (uint64_t)(uint32_t)(j_ + RS * i) * a.k_nb1 + (F::quant ? 0 : cc * 16);
    const uint32_t klds = lds_at(kt) + wave * 1024, clds = lds_at(cl) + wave * 256;
    auto fetch = [&](int t, int b) {
        const char * tile = kb + (uint64_t)((uint32_t)t * PA_SLOTS) * a.k_nb1;
        const char * src[CN];
        const int last = a.n_kv - 1 - t * PA_SLOTS;
#pragma unroll
        for (int i = 0; i < CN; i++) src[i] = tile + off[i];
        if (last < PA_SLOTS - 1) {
#pragma unroll
            for (int i = 0; i < CN; i++) if (j_ + RS * i > last) src[i] = tile + (uint64_t)(uint32_t)last * a.k_nb1 + (F::quant ? 0 : cc * 16);
        }
        if constexpr (F::quant) {
#pragma unroll
            for (int i = 0; i < CN; i++) { kr[i].load(src[i] + Chunk<TYPE>::at(cc)); kdr[i] = *(const uint16_t *)(src[i] + (cc >> 2) * F::block); }
        } else {
#pragma unroll
            for (int i = 0; i < CN; i++) dma16(src[i], klds + b * (PA_SLOTS * D * 2) + i * (PT * 16));
        }
        dma4(crow + (t * 2 & ~3), clds + b * (int)sizeof(cl[0]));
    };
    auto commit = [&](int b) {
        if constexpr (F::quant) {
#pragma unroll
            for (int i = 0; i < CN; i++) {
                *(v4i *)(kt[b] + lds_chunk<D>(j_ + RS * i, pos)) = kr[i].operand(cc);
                if ((pos & 3) == 0) kd[b][pos >> 2][j_ + RS * i] = kdr[i];
            }
        }
    };
    int t = split, b = 0;
    if (t < nt) { fetch(t, 0); commit(0); }
    if (S == 3 && t + ns < nt) fetch(t + ns, 1);
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int p = 0; p < QP; p++) arrived(qf[ks][p]);
    arrived(qe); arrived(slope);
    float m = -INFINITY, l = 0.0f;               // of this lane's row over this lane's slots (two lanes share a row)
    for (; t < nt; t += ns) {
        if (S == 2 || t + ns >= nt) wait_meet<0>();
        else wait_meet<CN + 1>();
        // tile t is there, and the place of the one before it is free
        const int ahead = t + (S - 1) * ns, bf = b == 0 ? S - 1 : b - 1;
        if (ahead < nt) fetch(ahead, bf);
        const uint32_t bytes = cl[b][wave][lane] >> (16 * (t & 1));
        const int c0 = bytes & 255, c1 = bytes >> 8 & 255;
        if (mine && __any((c0 | c1) != MASK_HIDDEN)) {
            v16f c[2], part;
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int i = 0; i < 16; i++) c[u][i] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const v4i k0 = *(const v4i *)(kt[b] + lds_chunk<D>(32 * u + lr, 2 * ks + lh));
                    if constexpr (F::quant) {
                        if (ks % 2 == 0) {
#pragma unroll
                            for (int i = 0; i < 16; i++) part[i] = 0.0f;
                        }
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) part = mfma32<F::bf>(k0, qf[ks][p], part);
                        if (ks % 2 == 1) fold_block(&kd[b][ks / 2][32 * u], lh, part, c[u]);
                    } else {
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) c[u] = mfma32<F::bf>(k0, qf[ks][p], c[u]);
                    }
                }
            }
            auto largest = [&]() {
                float x = c[0][0];
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x = max_or_nan(x, c[u][i]);
                return x;
            };
            float mx = F::quant ? 0.0f : largest();
            if constexpr (!F::quant) if (__builtin_expect(__any(mx != mx), 0)) {     // an infinity in a row of K (see finite); q comes from memory, in a short loop
                const uint16_t * qr = a.qparts + row * QP * D + 8 * lh;
#pragma unroll
                for (int u = 0; u < 2; u++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) c[u][i] = 0.0f;
#pragma unroll 1
                    for (int ks = 0; ks < KS; ks++) {
                        const v4i k0 = *(const v4i *)(kt[b] + lds_chunk<D>(32 * u + lr, 2 * ks + lh)), f = finite<F::bf>(k0);
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) c[u] = mfma32<F::bf>(p == 0 && 2 * ks + lh < a.d / 8 ? k0 : f, *(const v4i *)(qr + p * D + 16 * ks), c[u]);
                    }
                }
                mx = largest();
            }
            float sc = qe;
            if (CAP || !__all(c0 == MASK_ZERO && c1 == MASK_ZERO)) {
                tile_logits<CAP>(a, c[0], qe, slope, c0, mrow, m8, t * PA_SLOTS);
                tile_logits<CAP>(a, c[1], qe, slope, c1, mrow, m8, t * PA_SLOTS + 32);
                sc = 1.0f;
                mx = largest();
            } else if (F::quant) mx = largest();
            mx = max_or_nan(m, mx * sc);
            const float ms = mx == -INFINITY ? 0.0f : mx;
            l *= __builtin_amdgcn_exp2f(m - ms);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 16; i++) l += __builtin_amdgcn_exp2f(__builtin_fmaf(c[u][i], sc, -ms));
            m = mx;
        }
        if (S == 2 && ahead < nt) commit(bf);
        b = b == S - 1 ? 0 : b + 1;
    }
    const float mo = __shfl_xor(m, 32, 64), lo = __shfl_xor(l, 32, 64);
    const float M = fmaxf(m, mo), ms = M == -INFINITY ? 0.0f : M;
    const float L = l * __builtin_amdgcn_exp2f(m - ms) + lo * __builtin_amdgcn_exp2f(mo - ms);
    if (lh != 0 || r_ >= R) return;
    if (ns == 1) *(v2f *)&a.rowc[row].m = row_result(M, L);      // one slice: its statistics are the row's
    else *(v2f *)(a.stats + ((((int64_t)i3 * a.n_head_kv + hk) * ns + split) * R + r_) * 2) = v2f{M, L};
}

// several slices: their statistics of a row meet
__global__ void __launch_bounds__(PT)
prompt_rows_kernel(const MArgs a) {
    const int R = a.ratio * a.n_q, r = blockIdx.x * PT + threadIdx.x, hk = blockIdx.y, i3 = blockIdx.z;
    if (r >= R) return;
    const int64_t hrow = (int64_t)i3 * a.n_head_kv + hk;
    const v2f * st = (const v2f *)a.stats + hrow * a.nsplit * R + r;
    float M = -INFINITY, L = 0.0f;
    for (int s = 0; s < a.nsplit; s += 8) {
        v2f x[8];
        float mn = M;
#pragma unroll
        for (int i = 0; i < 8; i++) { x[i] = s + i < a.nsplit ? st[(int64_t)(s + i) * R] : v2f{-INFINITY, 0.0f}; mn = fmaxf(mn, x[i].x); }
        const float ms = mn == -INFINITY ? 0.0f : mn;
        L *= __builtin_amdgcn_exp2f(M - ms);
#pragma unroll
        for (int i = 0; i < 8; i++) L = __builtin_fmaf(x[i].y, __builtin_amdgcn_exp2f(x[i].x - ms), L);
        M = mn;
    }
    *(v2f *)&a.rowc[hrow * R + r].m = row_result(M, L);
}

// slots of a wave in the second pass: 64 where its K takes at most 64 registers so
template <int D> constexpr int prompt_ns() { return D <= 128 ? 2 : 1; }

template <int TYPE, int D, bool CAP>
__global__ void __launch_bounds__(PT, D <= 128 ? 2 : 1)
prompt_mass_kernel(const MArgs a) {
    typedef Fmt<TYPE> F;
    constexpr int NS = prompt_ns<D>();
    constexpr int KS = D / 16, QP = F::parts, S = D <= 128 ? 3 : 2;      // S: tiles in LDS
    constexpr int RS = PT / (D / 8), CP = PB_ROWS / RS, CN = QP * CP;       // passes of a part, of a tile
    __shared__ __attribute__((aligned(16))) uint8_t qt[S][QP][PB_ROWS * D * 2];
    __shared__ __attribute__((aligned(16))) float rc[S][PT / 64][64];       // RowC of the rows, twice
    __shared__ uint32_t cl[S][PT / 64][64];
    __shared__ __attribute__((aligned(16))) uint16_t kd[F::quant ? PT / 64 : 1][F::quant ? D / 32 : 1][32 * NS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, lh = lane >> 5;
    const int R = a.ratio * a.n_q, hk = blockIdx.y, i3 = blockIdx.z, chunk = blockIdx.x % a.nchunk;
    const int j0 = ((int)(turned() ? gridDim.x - 1 - blockIdx.x : blockIdx.x) / a.nchunk * 4 + wave) * 32 * NS;     // this wave's slots
    const int64_t base = ((int64_t)i3 * a.n_head_kv + hk) * R;
    const int nt = (R + PB_ROWS - 1) / PB_ROWS, nc = a.nchunk;
    const bool m8 = a.mask && (((uintptr_t)a.mask | (uintptr_t)a.m_nb1 | (uintptr_t)a.m_nb2 | (uintptr_t)a.m_nb3) & 7) == 0;
    const char * kb = a.k + hk * a.k_nb2 + i3 * a.k_nb3;

    const int pos = tid % (D / 8), x_ = tid / (D / 8), cc = pos ^ (x_ & swz<D>());
    const uint32_t qoff = (uint32_t)(x_ * QP * D + cc * 8) * 2, qlds = lds_at(qt) + wave * 1024, rlds = lds_at(rc) + wave * 256, clds = lds_at(cl) + wave * 256;
    auto fetch = [&](int t, int b) {                            // rows past the last one repeat it
        const int last = R - 1 - t * PB_ROWS;
        const char * tile = (const char *)a.qparts + (base + t * PB_ROWS) * (QP * D * 2), * rows = (const char *)(a.rowc + base + t * PB_ROWS);
        uint32_t o[CP], ro = 4 * (tid & 127);
        int r = t * PB_ROWS + lr;
#pragma unroll
        for (int i = 0; i < CP; i++) o[i] = qoff + RS * i * QP * D * 2;
        if (last < PB_ROWS - 1) {
#pragma unroll
            for (int i = 0; i < CP; i++) if (x_ + RS * i > last) o[i] = (uint32_t)(last * QP * D + cc * 8) * 2;
            if ((tid & 127) / 4 > last) ro = 16 * last + 4 * (tid & 3);
            if (lr > last) r = R - 1;
        }
#pragma unroll
        for (int i = 0; i < CN; i++) dma16(tile + o[i % CP] + i / CP * (D * 2), qlds + b * (int)sizeof(qt[0]) + i * (PT * 16));
        dma4(rows + ro, rlds + b * (int)sizeof(rc[0]));
        const int iq = m_query(a, r);
        dma4(class_row(a, iq, hk * a.ratio + r - iq * a.ratio, i3) + (j0 / 32 & ~3), clds + b * (int)sizeof(cl[0]));
    };
    int t = chunk, b = 0;
    if (t < nt) fetch(t, 0);
    if (S == 3 && t + nc < nt) fetch(t + nc, 1);

    // this wave's K rows, as the A operand holds them
    v4i kf[NS][KS];
#pragma unroll
    for (int u = 0; u < NS; u++) {
        const int j = j0 + 32 * u + lr;
        const char * krow = kb + (uint64_t)(uint32_t)(j < a.n_kv ? j : a.n_kv - 1) * a.k_nb1;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int cc = 2 * ks + lh < a.d / 8 ? 2 * ks + lh : a.d / 8 - 1;
            Chunk<TYPE> c;
            c.load(krow + Chunk<TYPE>::at(cc));
            kf[u][ks] = c.operand(cc);
            if constexpr (F::quant) if (ks % 2 == 0 && lh == 0) kd[wave][ks / 2][32 * u + lr] = *(const uint16_t *)(krow + (cc >> 2) * F::block);
        }
    }
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) arrived(kf[u][ks]);
    bool odd = false;                                           // an infinity in a row of K (see finite)
    if constexpr (!F::quant) {
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) { v4i x = kf[u][ks]; odd |= sanitize<F::bf>(x); }
        odd = __any(odd);
    }
    float acc[NS][16];
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[u][i] = 0.0f;

    for (; t < nt; t += nc) {
        if (S == 2 || t + nc >= nt) wait_meet<0>();
        else wait_meet<CN + 2>();
        const int ahead = t + (S - 1) * nc;
        if (ahead < nt) fetch(ahead, b == 0 ? S - 1 : b - 1);
        const uint32_t bytes = cl[b][wave][lane] >> (8 * (j0 / 32 & 3));
        int cu[NS], seen = MASK_HIDDEN;
        bool zero = !CAP;
#pragma unroll
        for (int u = 0; u < NS; u++) { cu[u] = bytes >> (8 * u) & 255; seen |= cu[u]; zero &= cu[u] == MASK_ZERO; }
        if (__any(seen != MASK_HIDDEN)) {
            RowC c4 = *(const RowC *)&rc[b][0][4 * lr];
            if (t * PB_ROWS + lr >= R) { c4.m = INFINITY; c4.inv = 0.0f; }      // weighs nothing
            v16f c[NS], part[NS];
            if (!F::quant && __builtin_expect(odd, 0)) {        // (K comes from memory again, in a short loop)
#pragma unroll
                for (int u = 0; u < NS; u++) {
                    const int j = j0 + 32 * u + lr;
                    const char * krow = kb + (uint64_t)(uint32_t)(j < a.n_kv ? j : a.n_kv - 1) * a.k_nb1;
#pragma unroll
                    for (int i = 0; i < 16; i++) c[u][i] = 0.0f;
#pragma unroll 1
                    for (int ks = 0; ks < KS; ks++) {
                        const bool in = 2 * ks + lh < a.d / 8;
                        const v4i k0 = *(const v4i *)(krow + 16 * (in ? 2 * ks + lh : 0)), f = finite<F::bf>(k0);
#pragma unroll
                        for (int p = QP - 1; p >= 0; p--) c[u] = mfma32<F::bf>(p == 0 && in ? k0 : f, *(const v4i *)(qt[b][p] + lds_chunk<D>(lr, 2 * ks + lh)), c[u]);
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) c[u][i] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    v4i q[QP];
                    if constexpr (F::quant) if (ks % 2 == 0) {
#pragma unroll
                        for (int u = 0; u < NS; u++)
#pragma unroll
                            for (int i = 0; i < 16; i++) part[u][i] = 0.0f;
                    }
#pragma unroll
                    for (int p = 0; p < QP; p++) q[p] = *(const v4i *)(qt[b][p] + lds_chunk<D>(lr, 2 * ks + lh));
#pragma unroll
                    for (int p = QP - 1; p >= 0; p--)
#pragma unroll
                        for (int u = 0; u < NS; u++) {
                            if constexpr (F::quant) part[u] = mfma32<F::bf>(kf[u][ks], q[p], part[u]);
                            else c[u] = mfma32<F::bf>(kf[u][ks], q[p], c[u]);
                        }
                    if constexpr (F::quant) if (ks % 2 == 1) {
#pragma unroll
                        for (int u = 0; u < NS; u++) fold_block(&kd[wave][ks / 2][32 * u], lh, part[u], c[u]);
                    }
                }
                // q is read two steps ahead of its products: beside the other branch the compiler reads it just before them (1024 x 1024, bf16, heads
                // of 256: 73 us for this pass, 61 so)
                if constexpr (!F::quant) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * QP, 0);
#pragma unroll
                    for (int ks = 0; ks < KS - 2; ks++) { __builtin_amdgcn_sched_group_barrier(0x8, QP * NS, 0); __builtin_amdgcn_sched_group_barrier(0x100, QP, 0); }
                    __builtin_amdgcn_sched_group_barrier(0x8, 2 * QP * NS, 0);
                }
            }
            float sc = c4.qe;
            if (!__all(zero)) {
                const int r = t * PB_ROWS + lr < R ? t * PB_ROWS + lr : R - 1, iq = m_query(a, r);
                const char * mrow = m_mask(a, iq, hk * a.ratio + r - iq * a.ratio, i3);
                int jm = j0;
                asm volatile("" : "+v"(jm));                    // (the comparisons of its slots with the last one would be kept through the loop)
#pragma unroll
                for (int u = 0; u < NS; u++) tile_logits<CAP>(a, c[u], sc, c4.slope, cu[u], mrow, m8, jm + 32 * u);
                sc = 1.0f;
            }
#pragma unroll
            for (int u = 0; u < NS; u++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[u][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(c[u][i], sc, -c4.m)), c4.inv, acc[u][i]);
        }
        b = b == S - 1 ? 0 : b + 1;
    }
    // over the 32 lanes (rows) of each half: 16 sums per tile.  One chunk: its sums are the weights
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float x = acc[u][i];
            x += dpp_f32<0xB1>(x); x += dpp_f32<0x4E>(x); x += dpp_f32<0x141>(x); x += dpp_f32<0x140>(x);
            x += __shfl_xor(x, 16, 64);
            const int j = j0 + 32 * u + 8 * (i >> 2) + 4 * lh + (i & 3);
            if (lr != 0 || j >= a.n_kv) continue;
            if (nc > 1) a.part[(((int64_t)i3 * a.n_head_kv + hk) * nc + chunk) * a.n_kv + j] = x;
            else mass_store(a, hk, i3, j, x);
        }
}

__global__ void __launch_bounds__(PT)
prompt_sum_kernel(const MArgs a) {
    const int j = blockIdx.x * PT + threadIdx.x, hk = blockIdx.y, i3 = blockIdx.z;
    if (j >= a.n_kv) return;
    const float * p = a.part + ((int64_t)i3 * a.n_head_kv + hk) * a.nchunk * a.n_kv + j;
    float t = 0.0f;
#pragma unroll 8
    for (int c = 0; c < a.nchunk; c++) t += p[(int64_t)c * a.n_kv];
    mass_store(a, hk, i3, j, t);
}

static int prompt_slots(int64_t d) {                     // slots of a workgroup in the second pass
    return step_d(d) <= 128 ? 256 : 128;
}
// Slices of the slots in the first pass: 512 workgroups, one round of two a CU (2047 x 2047: 67 us, with 1024 80, with 2048 87) and few
// slices to join (64: 8 us, 32: 5).  Small problems: a tile takes a workgroup that has the CU to itself 1.3 us, the launch that joins slices 4 -- up to 4
// tiles one slice, else down to one tile each (64 x 1024 x 32 heads, f16, the whole call: 26 us, with four tiles each 35,
// with two 29; 64 x 64: 21, 27, 23)
static int64_t prompt_splits(const mi355_fattn_args * p) {
    const int64_t R = p->n_head / p->n_head_kv * p->n_q, tiles = (p->n_kv + PA_SLOTS - 1) / PA_SLOTS, base = (R + PA_ROWS - 1) / PA_ROWS * p->n_head_kv * p->ne3;
    int64_t n = 512 / base, most = tiles <= 4 ? 1 : tiles;
    if (n > most) n = most;
    if (n > 32) n = 32;
    return n < 1 ? 1 : n;
}
// Slices of the rows in the second: likewise (2047 x 2047: 87 us, with 1024 93, with 768 104; 64 x 16384: 34, with 1024 38; both since 83, 32)
static int64_t prompt_chunks(const mi355_fattn_args * p) {
    const int64_t R = p->n_head / p->n_head_kv * p->n_q, tiles = (R + PB_ROWS - 1) / PB_ROWS;
    const int64_t ws = prompt_slots(p->d), base = (p->n_kv + ws - 1) / ws * p->n_head_kv * p->ne3;
    int64_t n = base > 0 ? 512 / base : 1, most = tiles <= 4 ? 1 : tiles;
    if (n > most) n = most;
    if (n > 32) n = 32;
    return n < 1 ? 1 : n;
}

// CAP (logit_softcap != 0) is a kernel of its own: the cap's code beside the other takes registers and 2 % of the time from q8_0 prompts without one
template <int TYPE, int D, bool CAP> static int prompt_launch(const MArgs & a, int ne3, hipStream_t s) {
    const int R = a.ratio * a.n_q, ws = 128 * prompt_ns<D>();
    const unsigned hk = (unsigned)a.n_head_kv, z = (unsigned)ne3;
    const int64_t slot_wgs = (a.n_kv + 1023) / 1024, query_wgs = a.mask ? (a.n_q + 3) / 4 : 1, class_wgs = slot_wgs * query_wgs * a.m_ne2 * a.m_ne3;
    const int64_t row_wgs = (R + 15) / 16, prep = class_wgs + row_wgs * hk * z;
    MI355_LAUNCH("attn_mass_prep", (prompt_prep_kernel<D, Fmt<TYPE>::bf>), dim3((unsigned)prep), dim3(PT), 0, s, a, (uint32_t)class_wgs, (uint32_t)slot_wgs,
                 (uint32_t)query_wgs, (uint32_t)row_wgs);
    MI355_CHECK_LAUNCH();
    MI355_LAUNCH("attn_mass_stats", (prompt_stats_kernel<TYPE, D, CAP>), dim3((unsigned)((R + PA_ROWS - 1) / PA_ROWS * a.nsplit), hk, z), dim3(PT), 0, s, a);
    MI355_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        MI355_LAUNCH("attn_mass_rows", prompt_rows_kernel, dim3((unsigned)((R + PT - 1) / PT), hk, z), dim3(PT), 0, s, a);
        MI355_CHECK_LAUNCH();
    }
    MI355_LAUNCH("attn_mass", (prompt_mass_kernel<TYPE, D, CAP>), dim3((unsigned)((a.n_kv + ws - 1) / ws * a.nchunk), hk, z), dim3(PT), 0, s, a);
    MI355_CHECK_LAUNCH();
    if (a.nchunk == 1) return MI355_OK;
    MI355_LAUNCH("attn_mass_sum", prompt_sum_kernel, dim3((unsigned)((a.n_kv + PT - 1) / PT), hk, z), dim3(PT), 0, s, a);
    MI355_CHECK_LAUNCH();
    return MI355_OK;
}
template <int TYPE> static int prompt_dispatch(const MArgs & a, int ne3, hipStream_t s) {
    if (a.n_kv == 0) return MI355_OK;
    const bool cap = a.logit_softcap != 0.0f;
    switch (step_d(a.d)) {
        case 64:  return cap ? prompt_launch<TYPE, 64, true>(a, ne3, s) : prompt_launch<TYPE, 64, false>(a, ne3, s);
        case 128: return cap ? prompt_launch<TYPE, 128, true>(a, ne3, s) : prompt_launch<TYPE, 128, false>(a, ne3, s);
    }
    return cap ? prompt_launch<TYPE, 256, true>(a, ne3, s) : prompt_launch<TYPE, 256, false>(a, ne3, s);
}

// steps: [statistics][partial rows of dst][logits]; prompts: [statistics][sums of the row chunks][row constants][parts of q][classes of the mask] (in floats)
struct WsParts { int64_t nsplit, nchunk, lpitch, stats, part, logits, rowc, q, cls; };
static int64_t class_pitch(int64_t n_kv) { return (n_kv + 511) / 512 * 16; }    // a byte per tile, whole workgroups of either pass
static WsParts mass_parts(const mi355_fattn_args * p, bool with_dst) {
    const int64_t rows = p->ne3 * p->n_head * p->n_q;
    WsParts w = {1, 1, 0, 0, 0, 0, 0, 0, 0};
    if (p->n_q > MI355_MASS_MAX_Q) {
        w.nsplit = prompt_splits(p);
        w.nchunk = prompt_chunks(p);
        w.stats = w.nsplit > 1 ? (w.nsplit * rows * 2 + 3) / 4 * 4 : 0;
        w.part = w.nchunk > 1 ? (p->ne3 * p->n_head_kv * w.nchunk * p->n_kv + 3) / 4 * 4 : 0;
        w.rowc = rows * 4;
        w.q = rows * step_d(p->d) / 2 * (p->type_k == MI355_TYPE_BF16 ? 3 : 2);
        w.cls = (p->mask ? p->m_ne2 * p->m_ne3 * p->n_q : 1) * class_pitch(p->n_kv) / 4;
    } else if (step_one(p)) {
        w.lpitch = (p->n_kv + 3) / 4 * 4;
        w.logits = rows * w.lpitch;
    } else {
        w.nsplit = step_splits(p);
        w.lpitch = (p->n_kv + 3) / 4 * 4;
        w.stats = (w.nsplit * rows * 2 + 3) / 4 * 4;
        w.part = with_dst ? w.nsplit * rows * step_d(p->d) : 0;
        w.logits = rows * w.lpitch;
    }
    return w;
}
static int64_t prep_workgroups(const mi355_fattn_args * p) {
    const int64_t classes = (p->n_kv + 1023) / 1024 * (p->mask ? (p->n_q + 3) / 4 * p->m_ne2 * p->m_ne3 : 1);
    return classes + (p->n_head / p->n_head_kv * p->n_q + 15) / 16 * p->n_head_kv * p->ne3;
}
// the shapes and types that both entry points take; what the workspace's size is formed from is bounded here, so its products stay within 64 bits
static int mass_shape(const mi355_fattn_args * p, bool with_dst) {
    const int64_t dv = p->dv ? p->dv : p->d;
    if (p->d < 8 || p->d > 256 || p->d % 8 != 0) return MI355_E_UNSUPPORTED;
    if (with_dst && (dv < 8 || dv > p->d || dv % 8 != 0)) return MI355_E_UNSUPPORTED;
    if (p->type_k != MI355_TYPE_F16 && p->type_k != MI355_TYPE_BF16 && p->type_k != MI355_TYPE_Q8_0 && p->type_k != MI355_TYPE_Q4_0) return MI355_E_TYPE;
    if (with_dst && p->type_v != p->type_k) return MI355_E_TYPE;
    const bool quant = p->type_k == MI355_TYPE_Q8_0 || p->type_k == MI355_TYPE_Q4_0;
    if (quant && (p->d % 32 != 0 || (with_dst && dv % 32 != 0))) return MI355_E_SHAPE;
    if (p->n_head < 1 || p->n_head > 65535 || p->n_head_kv < 1 || p->n_head % p->n_head_kv != 0 || p->n_q < 1 || p->n_q > 65535 || p->n_kv < 0 ||
        p->n_kv > (1 << 30) || p->ne3 < 1 || p->ne3 > 65535) return MI355_E_SHAPE;
    const int64_t ratio = p->n_head / p->n_head_kv;
    if (ratio * ratio * p->n_q > 0xffffffffll) return MI355_E_SHAPE;
    if (with_dst && p->n_q > MI355_MASS_MAX_Q) return MI355_E_UNSUPPORTED;
    if (p->mask && (p->m_ne2 < 1 || p->m_ne3 < 1 || p->m_ne2 > 65535 || p->m_ne3 > 65535 || p->m_ne2 * p->m_ne3 > 65535)) return MI355_E_SHAPE;
    // prompt_prep's grid: less than 2^32 threads, a workgroup of 256 for 16 rows of q or 4 x 1024 places of a mask
    if (p->n_q > MI355_MASS_MAX_Q && prep_workgroups(p) * PT > 0xffffffffll) return MI355_E_SHAPE;
    // steps keep a logit per (row, slot): more than 2^56 of them are no memory's size
    if (p->n_q <= MI355_MASS_MAX_Q && p->ne3 * p->n_head * p->n_q > (1ll << 56) / (p->n_kv + 4)) return MI355_E_SHAPE;
    return MI355_OK;
}
static int64_t mass_workspace(const mi355_fattn_args * p, bool with_dst) {
    if (!p || mass_shape(p, with_dst) != MI355_OK) return -1;
    const WsParts w = mass_parts(p, with_dst);
    return (w.stats + w.part + w.logits + w.rowc + w.q + w.cls) * 4;
}

static int mass_run(const mi355_fattn_args * p, const mi355_attn_mass_args * w, bool with_dst, void * workspace, int64_t workspace_bytes, void * stream) {
    if (!p || !w || !p->q || (p->n_kv > 0 && (!p->k || !w->mass_out)) || (with_dst && (!p->dst || (p->n_kv > 0 && !p->v)))) return MI355_E_NULL;
    const int shape = mass_shape(p, with_dst);
    if (shape != MI355_OK) return shape;
    const int64_t dv = p->dv ? p->dv : p->d, ratio = p->n_head / p->n_head_kv;
    const bool quant = p->type_k == MI355_TYPE_Q8_0 || p->type_k == MI355_TYPE_Q4_0;
    if (p->k_nb1 < 0 || p->k_nb1 > 0x7fffffff || (with_dst && (p->v_nb1 < 0 || p->v_nb1 > 0x7fffffff))) return MI355_E_SHAPE;
    const int64_t f32s = (int64_t)(uintptr_t)p->q | p->q_nb1 | p->q_nb2 | p->q_nb3 |
                         (with_dst ? (int64_t)(uintptr_t)p->dst | p->d_nb1 | p->d_nb2 | p->d_nb3 : 0) | (int64_t)(uintptr_t)workspace;
    int64_t cache = (int64_t)(uintptr_t)p->k | p->k_nb1 | p->k_nb2 | p->k_nb3;
    if (with_dst) cache |= (int64_t)(uintptr_t)p->v | p->v_nb1 | p->v_nb2 | p->v_nb3;
    const int64_t words = (int64_t)(uintptr_t)w->mass_in | w->in_nb2 | w->in_nb3 | (int64_t)(uintptr_t)w->mass_out | w->out_nb2 | w->out_nb3;
    const int64_t halves = p->mask ? (int64_t)(uintptr_t)p->mask | p->m_nb1 | p->m_nb2 | p->m_nb3 : 0;
    if ((f32s & 15) || (cache & (quant ? 1 : 15)) || (words & 3) || (halves & 1)) return MI355_E_ALIGN;
    if (w->mass_in && w->decay != 0.0f) {             // in place or apart: a shifted table would be read after other slots of it have been written
        const Span mi(w->mass_in, p->n_kv * 4, 1, 0, p->n_head_kv, w->in_nb2, p->ne3, w->in_nb3), mo(w->mass_out, p->n_kv * 4, 1, 0, p->n_head_kv, w->out_nb2, p->ne3, w->out_nb3);
        if (!mi.same(mo) && spans_meet(mi, mo)) return MI355_E_UNSUPPORTED;
    }
    const int64_t need = mass_workspace(p, with_dst);
    if (need > 0 && (!workspace || workspace_bytes < need)) return MI355_E_WORKSPACE;
    if (Span(w->mass_out, p->n_kv * 4, 1, 0, p->n_head_kv, w->out_nb2, p->ne3, w->out_nb3).folds() ||       // no place is written twice
        (with_dst && Span(p->dst, dv * 4, p->n_head, p->d_nb1, p->n_q, p->d_nb2, p->ne3, p->d_nb3).folds())) return MI355_E_UNSUPPORTED;

    MArgs a;
    a.q = (const char *)p->q; a.q_nb1 = p->q_nb1; a.q_nb2 = p->q_nb2; a.q_nb3 = p->q_nb3;
    a.k = (const char *)p->k; a.k_nb1 = (uint32_t)p->k_nb1; a.k_nb2 = p->k_nb2; a.k_nb3 = p->k_nb3;
    a.v = (const char *)p->v; a.v_nb1 = (uint32_t)p->v_nb1; a.v_nb2 = p->v_nb2; a.v_nb3 = p->v_nb3;
    a.mask = (const char *)p->mask; a.m_nb1 = p->m_nb1; a.m_nb2 = p->m_nb2; a.m_nb3 = p->m_nb3; a.m_ne2 = p->mask ? (int)p->m_ne2 : 1; a.m_ne3 = p->mask ? (int)p->m_ne3 : 1;
    a.ratio = (int)ratio; a.by_ratio = a.ratio > 1 ? (uint32_t)(((1ull << 32) + a.ratio - 1) / a.ratio) : 0;
    a.dst = with_dst ? (char *)p->dst : nullptr; a.d_nb1 = p->d_nb1; a.d_nb2 = p->d_nb2; a.d_nb3 = p->d_nb3;
    a.mass_in = w->decay != 0.0f ? (const char *)w->mass_in : nullptr; a.in_nb2 = w->in_nb2; a.in_nb3 = w->in_nb3;
    a.mass_out = (char *)w->mass_out; a.out_nb2 = w->out_nb2; a.out_nb3 = w->out_nb3;
    a.n_q = (int)p->n_q; a.n_kv = (int)p->n_kv; a.n_head_kv = (int)p->n_head_kv; a.d = (int)p->d; a.dv = (int)dv;
    a.scale = p->scale; a.max_bias = p->max_bias; a.logit_softcap = p->logit_softcap; a.decay = w->decay;
    a.n_head_log2 = 1u << (uint32_t)floorf(log2f((float)p->n_head));
    a.m0 = powf(2.0f, -(p->max_bias) / a.n_head_log2);
    a.m1 = powf(2.0f, -(p->max_bias / 2.0f) / a.n_head_log2);
    const WsParts parts = mass_parts(p, with_dst);
    a.one = p->n_q <= MI355_MASS_MAX_Q && step_one(p);
    a.nsplit = (int)parts.nsplit; a.nchunk = (int)parts.nchunk; a.lpitch = (int)parts.lpitch;
    a.stats = (float *)workspace;
    a.part = a.stats + parts.stats;
    a.logits = a.part + parts.part;
    a.rowc = (RowC *)(a.logits + parts.logits);
    a.qparts = (uint16_t *)(a.logits + parts.logits + parts.rowc);
    a.cls = (uint8_t *)(a.logits + parts.logits + parts.rowc + parts.q); a.cpitch = (int)class_pitch(p->n_kv);
    hipStream_t s = (hipStream_t)stream;
    if (p->n_q <= MI355_MASS_MAX_Q) switch (p->type_k) {
        case MI355_TYPE_F16:  return with_dst ? step_dispatch<MI355_TYPE_F16, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_F16, false>(a, (int)p->ne3, s);
        case MI355_TYPE_BF16: return with_dst ? step_dispatch<MI355_TYPE_BF16, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_BF16, false>(a, (int)p->ne3, s);
        case MI355_TYPE_Q8_0: return with_dst ? step_dispatch<MI355_TYPE_Q8_0, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_Q8_0, false>(a, (int)p->ne3, s);
        case MI355_TYPE_Q4_0: return with_dst ? step_dispatch<MI355_TYPE_Q4_0, true>(a, (int)p->ne3, s) : step_dispatch<MI355_TYPE_Q4_0, false>(a, (int)p->ne3, s);
    }
    switch (p->type_k) {
        case MI355_TYPE_F16:  return prompt_dispatch<MI355_TYPE_F16>(a, (int)p->ne3, s);
        case MI355_TYPE_BF16: return prompt_dispatch<MI355_TYPE_BF16>(a, (int)p->ne3, s);
        case MI355_TYPE_Q8_0: return prompt_dispatch<MI355_TYPE_Q8_0>(a, (int)p->ne3, s);
    }
    return prompt_dispatch<MI355_TYPE_Q4_0>(a, (int)p->ne3, s);
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
