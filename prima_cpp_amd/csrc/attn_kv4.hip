// attn_kv4.hip — attention over pages held in 4 bits: causal, with a sliding window and first tokens that stay visible.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp2(cf q k_j - max), over the j that the query sees; one pass over the keys with the running maximum and sum, both products on the f16 matrix cores.
// Keys and values become f16 on their way to the products: a pair of codes is masked out of a word over the bits of 1024, less 1032, times the scale - 3.25 operations for two values (the words are
// ordered so that a mask gives a pair that an operand wants). Queries are brought to [1, 2) by a power of two per row: exact for bf16 values down to 2^-17 of their row's largest, smaller ones are off
// by 2^-25 of it at most (f16's last step). Probabilities are held times 2^8, so that f16 has its steps of 2^-11 down to p = 2^-22. With bf16 rows they are single f16, an eighth of the step of the
// output that they make: the error of long and prompt attention against 64 bits is 0.00166 .. 0.00168 of the values, 0.00165 .. 0.00167 of it the output's own rounding; as pairs of f16 a prompt of
// 4096 tokens would take 406 us instead of 322 (in a graph), 48 tokens 89 instead of 84. WIDE (32-bit rows) holds queries and probabilities as pairs and makes two products of each.
// S^T = K Q^T is computed with the key rows permuted so that a lane's score registers are its P operand of O^T = V^T P^T.
//   few    16 or 32 columns (tokens x query heads of a KV head) per workgroup, 32 keys per wave and step, keys split over waves and workgroups: bound by memory, short prompt portions by the way
//          through one step. 48 tokens of 64 heads behind 3300 .. 8203 keys 74 us (329 MB, 4.4 TB/s), one of 32 heads behind 131100 37 us (151 MB), 16 x 4 of 28 heads in a window of 4096 24 us; a large copy reaches 4.9 TB/s here
//   tiles  128 columns per workgroup, a page at a time through LDS, where it is made f16 once for all four waves: bound by the matrix cores, which run at 1.1 .. 1.3 PFLOP/s under load.
//          4096 tokens of 32 heads behind 2011: 311 .. 318 us, 857 .. 876 TFLOP/s (a large f16 product of the library 1110). 32-bit rows of 256 spill 88 registers: 512 tokens of 16 + 4 heads 63 us, bf16 37
//   join   the partial sums of split keys
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include "../../include/prima_mi355.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -3e38f;                             // running maximum before the first visible key
constexpr float FAR = 16777216.0f;                         // beyond 2^24 a maximum is rounded by more than 1 (2^15 is the last power that f16 has): scores are rounded like it, then it is taken off
constexpr float HELD = 8.0f, SLACK = 6.0f;                 // probabilities are held times 2^HELD; the running maximum may lag by SLACK (2^14 < 65504), sums are seldom rescaled

// N words (N halves) that lie side by side, a multiple of 4 N (2 N) bytes into a slab
template <int N> __device__ __forceinline__ void ld_words(const PM_G char * p, uint32_t * w) {
    if constexpr (N == 2) { const u32x2 t = *(const PM_G u32x2 *) p; w[0] = t.x; w[1] = t.y; }
    else if constexpr (N == 3) { const u32x3 t = *(const PM_G u32x3 *) p; w[0] = t.x; w[1] = t.y; w[2] = t.z; }
    else if constexpr (N == 4) { const u32x4 t = *(const PM_G u32x4 *) p; w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
    else { ld_words<N / 2>(p, w); ld_words<N / 2>(p + 2 * N, w + N / 2); }
}
template <int N> __device__ __forceinline__ void ld_halves(const PM_G char * p, uint32_t * w) {
    if constexpr (N == 3) {
        const PM_G uint16_t * h = (const PM_G uint16_t *) p;
        w[0] = h[0] | (uint32_t) h[1] << 16; w[1] = h[2];
    } else if constexpr (N == 2) w[0] = *(const PM_G uint32_t *) p;
    else ld_words<N / 2>(p, w);
}
__device__ __forceinline__ f16x2 half_of(const uint32_t * w, int i) {      // value i of packed halves, twice
    const f16x2 t = __builtin_bit_cast(f16x2, w[i >> 1]);
    return i & 1 ? f16x2{t.y, t.y} : f16x2{t.x, t.x};
}
// The four pairs of codes of a word, less 8: those at nibbles 0 and 2 over the bits of 1024, those at 1 and 3 are 1024 + 16 code. The masks are held in registers, one of them a vector
// register: of two constants that it can see the compiler makes two operations instead of one v_and_or_b32.
struct pm_masks { uint32_t even, odd, bits; };
__device__ __forceinline__ pm_masks masks() {
    pm_masks m{0x000f000fu, 0x00f000f0u, 0x64006400u};
    asm("" : "+s"(m.even), "+s"(m.odd), "+v"(m.bits));
    return m;
}
__device__ __forceinline__ void codes(uint32_t w, const pm_masks & m, f16x2 * n) {
    const uint32_t u = w >> 8;
    const f16x2 zero = {(_Float16) -1032.0f, (_Float16) -1032.0f}, part = {(_Float16) 0.0625f, (_Float16) 0.0625f}, less = {(_Float16) -72.0f, (_Float16) -72.0f};
    n[0] = __builtin_bit_cast(f16x2, (w & m.even) | m.bits) + zero;
    n[1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & m.odd) | m.bits), part, less);
    n[2] = __builtin_bit_cast(f16x2, (u & m.even) | m.bits) + zero;
    n[3] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (u & m.odd) | m.bits), part, less);
}
__device__ __forceinline__ f16x8 eight(f16x2 a, f16x2 b, f16x2 c, f16x2 d) { return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; }
// scales beyond what the cache store makes (8188: its codes stay finite), NaN and infinities become 0; bits 0, 1: which
__device__ __forceinline__ uint32_t finite(uint32_t & s) {
    const uint32_t lo = (s & 0x7fffu) > 0x6fffu, hi = (s & 0x7fffffffu) > 0x6fffffffu;
    s &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    return lo | hi << 1;
}
template <typename T> __device__ __forceinline__ void st_out(T * p, f32x4 v) {
    if constexpr (sizeof(T) == 2) *(PM_G u16x4 *) p = u16x4{f2bf(v.x), f2bf(v.y), f2bf(v.z), f2bf(v.w)};
    else *(PM_G f32x4 *) p = v;
}

// eight values of a query row as operands, times a power of two
template <typename T> __device__ __forceinline__ void ld_query(const T * p, float * x) {
    if constexpr (sizeof(T) == 2) {
        const u32x4 t = *(const PM_G u32x4 *) p;
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[2 * j] = __builtin_bit_cast(float, t[j] << 16); x[2 * j + 1] = __builtin_bit_cast(float, t[j] & 0xffff0000u); }
    } else {
        const f32x4 a = *(const PM_G f32x4 *) p, b = *(const PM_G f32x4 *) (p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = a[j]; x[j + 4] = b[j]; }
    }
}
__device__ __forceinline__ void split_f16(const float * x, f16x8 & hi, f16x8 & lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { hi[j] = (_Float16) x[j]; lo[j] = (_Float16) (x[j] - (float) hi[j]); }
}
// 2^-e with the sign of scale for a row whose largest magnitude is in [2^e, 2^(e + 1)); cf = |scale| log2(e) 2^e, up to 2^100: scores (below 2^25) differ by 2^-48 at the least.
// NaN for a row with an infinity: whatever keys it meets its softmax is NaN, but scores of nothing but -inf would pass for keys that are hidden
__device__ __forceinline__ float row_factor(float most, float scale, float & cf) {
    int e = (int) (__builtin_bit_cast(uint32_t, most) >> 23 & 255) - 127;
    const bool finite = e < 128;
    e = finite ? e : 0;                                    // (-127: zeros, and numbers below 2^-126)
    cf = fminf(fmaxf(fabsf(scale) * ldexpf(1.0f, e) * LOG2E, 1e-30f), 0x1p100f);      // (in this order nothing on the way leaves 32 bits that the end does not)
    return finite ? copysignf(ldexpf(1.0f, -e), scale) : NAN;
}

// what the columns of a tile see together: pages [0, front) and from p0 on, `count` in all
struct pm_seen { int lo, hi, front, p0, count; };
__device__ __forceinline__ pm_seen seen_by(const pm_kv4_cache & c, const pm_kv4_attn & a, int pos, int n) {
    pm_seen s{pos, pos + n - 1, 0, 0, 0};
    if (pos < 0) return s;
    const int from = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, last = s.hi / PM_PAGE < c.table_ld ? s.hi / PM_PAGE : c.table_ld - 1;
    s.p0 = from / PM_PAGE;
    const int f = (int) (((int64_t) a.first + PM_PAGE - 1) / PM_PAGE);
    s.front = s.p0 < f ? s.p0 : f;
    if (s.front > c.table_ld) s.front = c.table_ld;
    s.count = s.front + (last >= s.p0 ? last - s.p0 + 1 : 0);
    return s;
}
__device__ __forceinline__ int page_at(const pm_seen & s, int i) { return i < s.front ? i : s.p0 + i - s.front; }

// ---- few columns ------------------------------------------------------------------------------------------------------------
constexpr int FW = 8, STAGES = 2;                          // waves of a workgroup; steps of a wave whose codes have a place in LDS
// 32 keys in LDS: key codes (rows of 16 NB bytes), value codes, key scales, value scales [NB][32]
template <int NB> struct pm_step {
    static constexpr int V = 512 * NB, KS = 1024 * NB, VS = 1088 * NB, BYTES = 1152 * NB;
    static constexpr int WIDE_LOADS = (512 * NB + 1023) / 1024, NARROW_LOADS = (64 * NB + 255) / 256, LOADS = 2 * (WIDE_LOADS + NARROW_LOADS);
};
// LDS <- 64 x 16 (64 x 4) bytes like pm_dma16, for codes that are read once
__device__ __forceinline__ void dma16(const void * base, uint32_t voff, uint32_t dst) {
    unsigned keep;
    dst = (uint32_t) __builtin_amdgcn_readfirstlane((int) dst);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(uniform_ptr((char *) base)), "s"(dst) : "memory");
}
__device__ __forceinline__ void dma4(const void * base, uint32_t voff, uint32_t dst) {
    unsigned keep;
    dst = (uint32_t) __builtin_amdgcn_readfirstlane((int) dst);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2 nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(uniform_ptr((char *) base)), "s"(dst) : "memory");
}
template <int N> __device__ __forceinline__ void lds_words(const char * p, uint32_t * w) {
    if constexpr (N == 1) w[0] = *(const uint32_t *) p;
    else if constexpr (N == 2) { const u32x2 t = *(const u32x2 *) p; w[0] = t.x; w[1] = t.y; }
    else if constexpr (N == 4) { const u32x4 t = *(const u32x4 *) p; w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
    else if constexpr (N == 3) { w[0] = ((const uint32_t *) p)[0]; w[1] = ((const uint32_t *) p)[1]; w[2] = ((const uint32_t *) p)[2]; }
    else { lds_words<N / 2>(p, w); lds_words<N / 2>(p + 2 * N, w + N / 2); }
}
template <int NB> __device__ __forceinline__ void lds_halves(const char * p, uint32_t * w) {
    if constexpr (NB == 3) { const uint16_t * h = (const uint16_t *) p; w[0] = h[0] | (uint32_t) h[1] << 16; w[1] = h[2]; }
    else lds_words<NB / 2>(p, w);
}

// consecutive numbers for the workgroups of an XCD (workgroup i starts on XCD i mod 8)
__device__ __forceinline__ uint32_t swizzled() {
    const uint32_t n = gridDim.x, x = blockIdx.x & 7, q = n >> 3, r = n & 7;
    return x * q + (x < r ? x : r) + (blockIdx.x >> 3);
}
// CT column tiles of 16 per workgroup share the keys' way from codes to f16; `launched` workgroups take the columns of a tile
template <typename T, int NB, bool WIDE, int CT> __global__ __launch_bounds__(FW * 64, NB <= 4 && CT == 1 && !WIDE ? 4 : 2) void few_kernel(pm_kv4_cache c, pm_kv4_attn a, int launched, int passes, int splits) {
    constexpr int D = NB * 32, VT = D / 16, LD = D + 4, COLS = 16 * CT;
    typedef pm_kv4_slab<NB> S;
    typedef pm_step<NB> Q;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [FW][STAGES] steps; then [FW][16][LD] sums
    float * acc_l = (float *) lds;
    __shared__ float m_l[FW][16], l_l[FW][16];
    const uint32_t id = swizzled();
    const int G = c.G, R = a.H / G, g = id % G, s = id / G / launched % splits, at = id / G / launched / splits;
    const int32_t * tile = uniform_const_ptr(a.tiles) + (size_t) at * 4;
    const int row0 = tile[0], seq = tile[3], pos0 = tile[2] < 0x7fffff00 ? tile[2] : 0x7fffff00, n = tile[1] < a.tile_tokens ? tile[1] : a.tile_tokens;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    // (tiles may have more columns than they have on the average, for which the launch is made: with CT > 1 a workgroup takes the further ones too. Workgroups without work are no way
    // out: each waits for its LDS behind those that work)
    int pass = id / G % launched;
    if (n < 1 || pass * COLS >= n * R) return;             // (what a tile's count is times R may leave 32 bits where it is negative)
    do {
    const size_t slot = ((size_t) at * passes + pass) * G + g;
    const int col0 = pass * COLS, left = n * R - col0, cols = left < COLS ? left : COLS;
    const int t0 = col0 / R, tn = (col0 + cols - 1) / R - t0 + 1;          // tokens of the columns
    const pm_seen see = seen_by(c, a, pos0 < 0 ? -1 : pos0 + t0, tn);
    const int per = (see.count + splits - 1) / splits, end = 2 * ((s + 1) * per < see.count ? (s + 1) * per : see.count);
    const bool known = (unsigned) seq < (unsigned) c.n_seq;
    const int32_t * table = uniform_const_ptr(c.table) + (size_t) (known ? seq : 0) * c.table_ld;
    const char * head = c.pages + (size_t) g * S::BYTES;
    auto page_of = [&](int i) __attribute__((always_inline)) { if (!known || i >= end) return -1; const int p = table[page_at(see, i >> 1)]; return (unsigned) p < (unsigned) c.n_pages ? p : -1; };
    const uint32_t krow = 8 * (lr >> 2) + (lr & 3);        // key of score row lr in the first 16 of a step (the second: + 4)
    // Codes go from memory to LDS in whole lines and from there to the lanes that want them (straight to registers every lane wants 16 bytes of another line of 64, and a step on its way costs
    // 36 registers: no slower with 4 waves of 128 registers, but 8 of them do not fit). Rows whose pieces would meet in a bank are turned against each other.
    constexpr int TURN = NB % 4 ? 0 : NB / 4;
    char * const ring = lds + wave * STAGES * Q::BYTES;
    const uint32_t ring_at = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) char *) lds + wave * STAGES * Q::BYTES;
    const uint32_t at_k = krow * 16 * NB + (TURN ? (lg ^ (krow >> 3 & 3)) : lg) * 4 * NB;
    auto load = [&](int i, int page, int stage) __attribute__((always_inline)) {
        const char * slab = uniform_ptr((char *) head + (size_t) (page < 0 ? 0 : page) * G * S::BYTES);      // (what is not there is read from page 0 and left alone)
        const char * k = slab + S::K + (i & 1) * 512 * NB, * v = slab + S::V + (i & 1) * 512 * NB, * ks = slab + S::KS + (i & 1) * 64 * NB, * vs = slab + S::VS + (i & 1) * 64;
        const uint32_t to = ring_at + stage * Q::BYTES;
#pragma unroll
        for (int j = 0; j < Q::WIDE_LOADS; ++j) {
            const uint32_t o = lane * 16 + j * 1024, row = o / (16 * NB);
            if (o < 512 * NB) { dma16(k, TURN ? o ^ (row >> 3 & 3) * (16 * TURN) : o, to + j * 1024); dma16(v, o, to + Q::V + j * 1024); }
        }
#pragma unroll
        for (int j = 0; j < Q::NARROW_LOADS; ++j) {
            const uint32_t o = lane * 4 + j * 256;
            if (o < 64 * NB) { dma4(ks, o, to + Q::KS + j * 256); dma4(vs, (o >> 6) * (PM_PAGE * 2) + (o & 63), to + Q::VS + j * 256); }
        }
    };
    const pm_masks mk = masks();
    int i = 2 * s * per + wave, page = page_of(i), next = page_of(i + FW), stage = 0;
    if (i < end) load(i, page, 0);
    if (i + FW < end) load(i + FW, next, 1);

    f16x8 qh[CT][NB], ql[WIDE ? CT : 1][NB];
    f32x4 acc[CT][VT];
    float cf[CT], m[CT], l[CT];
    int pos[CT];
    bool far = false;
#pragma unroll
    for (int u = 0; u < CT; ++u) {
        const int col = u * 16 + lr, tok = (col0 + col) / R, row = row0 + tok, h = g * R + (col0 + col) % R;
        const bool on = col < cols && (unsigned) row < (unsigned) a.n_tokens;
        pos[u] = col < cols && pos0 >= 0 ? pos0 + tok : -1;
        float x[NB][8], most = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
            if (on) ld_query<T>((const T *) a.q + (size_t) row * a.ldq + h * D + b * 32 + lg * 8, x[b]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[b][j]));
        }
        most = fmaxf(most, __shfl_xor(most, 16)); most = fmaxf(most, __shfl_xor(most, 32));
        const float f = row_factor(most, a.scale, cf[u]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] *= f;
            f16x8 lo;
            split_f16(x[b], qh[u][b], lo);
            if (WIDE) ql[u][b] = lo;
        }
#pragma unroll
        for (int t = 0; t < VT; ++t) acc[u][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[u] = NONE; l[u] = 0.0f;
    }
    for (; i < end; i += FW) {
        const int after = page_of(i + 2 * FW);
        if (i + FW < end) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(Q::LOADS) : "memory");      // (a wave's loads come back in their order)
        else pm_vm_drain();
        const char * x = ring + stage * Q::BYTES;
        const int k0 = page_at(see, i >> 1) * PM_PAGE + (i & 1) * 32, key0 = k0 + lg * 8;      // the lane's eight keys
        f32x4 s0[CT], s1[CT];
#pragma unroll
        for (int u = 0; u < CT; ++u) s0[u] = s1[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t xk[2][NB], xs[2][(NB + 1) / 2], xv[2][NB], vs[NB][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) { lds_words<NB>(x + at_k + b * 64 * NB, xk[b]); lds_halves<NB>(x + Q::KS + (krow + 4 * b) * 2 * NB, xs[b]); }
#pragma unroll
        for (int b = 0; b < 2; ++b) lds_words<NB>(x + Q::V + (2 * lg + b) * 64 * NB + lr * 4 * NB, xv[b]);
#pragma unroll
        for (int w = 0; w < NB; ++w) lds_words<4>(x + Q::VS + w * 64 + lg * 16, vs[w]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const f16x2 sa = half_of(xs[0], b), sb = half_of(xs[1], b);
            f16x2 na[4], nb[4];
            codes(xk[0][b], mk, na); codes(xk[1][b], mk, nb);
            const f16x8 ka = eight(na[0] * sa, na[1] * sa, na[2] * sa, na[3] * sa), kb = eight(nb[0] * sb, nb[1] * sb, nb[2] * sb, nb[3] * sb);
#pragma unroll
            for (int u = 0; u < CT; ++u) {
                s0[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[u][b], s0[u], 0, 0, 0);
                s1[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qh[u][b], s1[u], 0, 0, 0);
                if (WIDE) { s0[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[u][b], s0[u], 0, 0, 0); s1[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, ql[u][b], s1[u], 0, 0, 0); }
            }
        }
        // a step that not every column sees whole: hidden keys count nothing, whatever their slots hold
        const bool whole = page >= 0 && k0 + 31 <= see.lo && !(a.window > 0 && k0 <= see.hi - a.window);
        uint32_t bad = 0;
        if (!whole) {
            asm volatile("");                              // (a branch: as selects this would cost every step as much as the products' operands)
#pragma unroll
            for (int w = 0; w < NB; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) bad |= finite(vs[w][j]) << 2 * j;
        }
        f16x8 ph[CT], pl[CT];
#pragma unroll
        for (int u = 0; u < CT; ++u) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = j < 4 ? s0[u][j & 3] : s1[u][j & 3];
            if (!whole) {
                asm volatile("");
                const int last = page < 0 ? -1 : pos[u], low = a.window > 0 ? pos[u] - a.window + 1 : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = key0 + j;
                    const bool ok = key <= last && (key >= low || key < a.first);
                    f[j] = ok ? (bad >> j & 1 ? NAN : f[j]) : -INFINITY;
                }
            }
            float mx = f[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx = fmaxf(mx, f[j]);
            mx = fmaxf(mx, __shfl_xor(mx, 16)); mx = fmaxf(mx, __shfl_xor(mx, 32));
            mx = fmaxf(mx * cf[u], NONE);
            if (__any(mx > m[u] + SLACK)) {
                const float mn = fmaxf(m[u], mx), corr = __builtin_amdgcn_exp2f(m[u] - mn);
                m[u] = mn; l[u] *= corr;
                far |= __any(fabsf(mn) > FAR && mn > NONE);
#pragma unroll
                for (int t = 0; t < VT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[u][t][e] *= corr;
            }
            float k = cf[u], mo = HELD - m[u];
            if (far) {
                asm volatile("");
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = f[j] * k - m[u];
                k = 1.0f; mo = HELD;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) { f[j] = __builtin_amdgcn_exp2f(fmaf(f[j], k, mo)); l[u] += f[j]; }
            split_f16(f, ph[u], pl[u]);
        }
#pragma unroll
        for (int w = 0; w < NB; ++w) {
            f16x2 sc[4], na[4], nb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[j] = __builtin_bit_cast(f16x2, vs[w][j]);
            codes(xv[0][w], mk, na); codes(xv[1][w], mk, nb);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f16x8 v = eight(na[h] * sc[0], na[h + 2] * sc[1], nb[h] * sc[2], nb[h + 2] * sc[3]);
#pragma unroll
                for (int u = 0; u < CT; ++u) {
                    acc[u][2 * w + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[u], acc[u][2 * w + h], 0, 0, 0);
                    if (WIDE) acc[u][2 * w + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[u], acc[u][2 * w + h], 0, 0, 0);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the stage is read: it may be written)
        if (i + 2 * FW < end) load(i + 2 * FW, after, stage);
        page = next; next = after; stage ^= 1;
    }
    __syncthreads();                                       // (the rings' LDS is the sums')
    auto store = [&](int col, int d, f32x4 o) {
        const int row = row0 + (col0 + col) / R;
        if ((unsigned) row < (unsigned) a.n_tokens) st_out((T *) a.out + (size_t) row * a.ldo + (g * R + (col0 + col) % R) * D + d, o);
    };
    float * part = a.work + slot * splits * COLS * (D + 2);
#pragma unroll
    for (int u = 0; u < CT; ++u) {
        const int have = cols - u * 16 < 16 ? cols - u * 16 : 16;          // (may be none)
        if (u) __syncthreads();
        l[u] += __shfl_xor(l[u], 16); l[u] += __shfl_xor(l[u], 32);
        if (lr < have) {
#pragma unroll
            for (int t = 0; t < VT; ++t) *(f32x4 *) (acc_l + (wave * 16 + lr) * LD + t * 16 + lg * 4) = acc[u][t];
            if (lg == 0) { m_l[wave][lr] = m[u]; l_l[wave][lr] = l[u]; }
        }
        __syncthreads();
        for (int o = threadIdx.x; o < have * (D / 4); o += FW * 64) {
            const int col = o / (D / 4), d = o % (D / 4) * 4;
            float M = NONE, sum = 0.0f;
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < FW; ++w) M = fmaxf(M, m_l[w][col]);
#pragma unroll
            for (int w = 0; w < FW; ++w) { const float f = __builtin_amdgcn_exp2f(m_l[w][col] - M); v += *(const f32x4 *) (acc_l + (w * 16 + col) * LD + d) * f; sum += l_l[w][col] * f; }
            if (splits == 1) store(u * 16 + col, d, v * (sum == 0.0f ? 0.0f : 1.0f / sum));
            else {
                *(PM_G f32x4 *) (part + (size_t) (s * COLS + u * 16 + col) * D + d) = v;
                if (d == 0) *(PM_G f32x2 *) (part + (size_t) splits * COLS * D + (s * COLS + u * 16 + col) * 2) = f32x2{M, sum};
            }
        }
    }
    __syncthreads();
    pass += launched;
    } while (CT > 1 && pass * COLS < n * R);
}

// ---- prompts ----------------------------------------------------------------------------------------------------------------
constexpr int AHEAD = 4;                                   // operands on their way from LDS
constexpr int TC = 128;                                    // columns of a tile: 32 per wave

template <typename T, int NB, bool WIDE> __global__ __launch_bounds__(256, NB <= 4 ? 2 : 1) void tiles_kernel(pm_kv4_cache c, pm_kv4_attn a, int splits) {
    constexpr int D = NB * 32, KS = D / 16, VT = D / 32, KL = D * 2 + 16, VL = PM_PAGE * 2 + 16;      // LDS rows are an odd number of 16-byte pieces: no bank is asked twice
    typedef pm_kv4_slab<NB> S;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // two pages: K [64][KL], V^T [D][VL]
    constexpr int STAGE = PM_PAGE * KL + D * VL;
    __shared__ __attribute__((aligned(16))) uint8_t bad_l[2][16];
    const int G = c.G, R = a.H / G, g = blockIdx.x % G, s = blockIdx.y;
    const int at = a.n_tiles - 1 - (int) (blockIdx.x / G);                // (later tiles see more keys: they start first)
    const size_t slot = (size_t) at * G + g;
    const int32_t * tile = uniform_const_ptr(a.tiles) + (size_t) at * 4;
    const int row0 = tile[0], seq = tile[3], pos0 = tile[2] < 0x7fffff00 ? tile[2] : 0x7fffff00, n = tile[1] < a.tile_tokens ? tile[1] : a.tile_tokens;
    if (n < 1) return;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 31, hf = lane >> 5, col = wave * 32 + lr, cols = n * R;
    const int ct = col < cols ? col / R : 0, ch = g * R + (col < cols ? col % R : 0), row = row0 + ct;
    const bool on = col < cols && (unsigned) row < (unsigned) a.n_tokens;
    const pm_seen see = seen_by(c, a, pos0, n);
    const int pos = col < cols && pos0 >= 0 ? pos0 + ct : -1, low = a.window > 0 ? pos - a.window + 1 : 0;
    const int w_hi = pos0 + ((wave * 32 + 31 < cols ? wave * 32 + 31 : cols - 1) / R);                    // last position of the wave's columns
    const bool w_on = wave * 32 < cols;
    const int per = (see.count + splits - 1) / splits, begin = s * per, end = begin + per < see.count ? begin + per : see.count;
    const bool known = (unsigned) seq < (unsigned) c.n_seq;
    const int32_t * table = uniform_const_ptr(c.table) + (size_t) (known ? seq : 0) * c.table_ld;
    const char * head = c.pages + (size_t) g * S::BYTES;
    auto page_of = [&](int i) __attribute__((always_inline)) { if (!known || i >= end) return -1; const int p = table[page_at(see, i)]; return (unsigned) p < (unsigned) c.n_pages ? p : -1; };
    // a page on its way: thread t has the codes of key row t / 4, dimensions 8 (t % 4) .. + 7 of each block, and of token quad t / 16, dimensions n and n + 16 of each block, n = t % 16
    const int kr = threadIdx.x >> 2, kg = threadIdx.x & 3, vq = threadIdx.x >> 4, vn = threadIdx.x & 15;
    const pm_masks mk = masks();
    uint32_t xk[NB], xks[(NB + 1) / 2], xv[NB], xvs[NB][2];
    auto load = [&](int page) __attribute__((always_inline)) {             // (what is not there is read from page 0 and hidden)
        const PM_G char * slab = (const PM_G char *) uniform_ptr((char *) head + (size_t) (page < 0 ? 0 : page) * G * S::BYTES);
        ld_words<NB>(slab + S::K + (uint32_t) (kr * 16 * NB + kg * 4 * NB), xk);
        ld_halves<NB>(slab + S::KS + (uint32_t) (kr * 2 * NB), xks);
        ld_words<NB>(slab + S::V + (uint32_t) (vq * 64 * NB + vn * 4 * NB), xv);
#pragma unroll
        for (int w = 0; w < NB; ++w) ld_words<2>(slab + S::VS + w * PM_PAGE * 2 + (uint32_t) (vq * 8), xvs[w]);
    };
    // every column sees the page whole; else scales that are not finite are taken out of it
    auto whole = [&](int i, int page) __attribute__((always_inline)) { const int key0 = page_at(see, i) * PM_PAGE; return page >= 0 && key0 + PM_PAGE - 1 <= see.lo && !(a.window > 0 && key0 <= see.hi - a.window); };
    auto clean = [&](int stage) __attribute__((always_inline)) {
        uint32_t bad = 0;
#pragma unroll
        for (int w = 0; w < NB; ++w) bad |= finite(xvs[w][0]) | finite(xvs[w][1]) << 2;
        if (vn == 0) bad_l[stage][vq] = (uint8_t) bad;
    };
    // the page in registers as f16, in 4 NB pieces: key block b in pieces 2 b and 2 b + 1 (codes; scale and store), value block b in 2 NB + 2 b and the one behind it
    f16x2 half_done[4];
    auto expand = [&](int piece, int stage) __attribute__((always_inline)) {
        const int b = piece / 2 % NB;
        const bool val = piece >= 2 * NB;
        if (piece % 2 == 0) { codes(val ? xv[b] : xk[b], mk, half_done); return; }
        char * k_l = lds + stage * STAGE, * v_l = k_l + PM_PAGE * KL;
        const f16x2 * n = half_done;
        if (!val) {
            const f16x2 sc = half_of(xks, b);
            *(f16x8 *) (k_l + kr * KL + (b * 4 + kg) * 16) = eight(n[0] * sc, n[1] * sc, n[2] * sc, n[3] * sc);
        } else {
            const f16x2 s0 = __builtin_bit_cast(f16x2, xvs[b][0]), s1 = __builtin_bit_cast(f16x2, xvs[b][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *(u32x2 *) (v_l + (b * 32 + h * 16 + vn) * VL + vq * 8) = u32x2{__builtin_bit_cast(uint32_t, n[h] * s0), __builtin_bit_cast(uint32_t, n[h + 2] * s1)};
        }
    };
    auto expand_all = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4 * NB; ++q) expand(q, stage);
    };
    int page = page_of(begin), next = page_of(begin + 1);
    load(page);

    f16x8 qh[KS], ql[KS];
    float cf;
    {
        float x[KS][8], most = 0.0f;
#pragma unroll
        for (int b = 0; b < KS; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
            if (on) ld_query<T>((const T *) a.q + (size_t) row * a.ldq + ch * D + b * 16 + hf * 8, x[b]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[b][j]));
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        const float f = row_factor(most, a.scale, cf);
#pragma unroll
        for (int b = 0; b < KS; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] *= f;
            split_f16(x[b], qh[b], ql[b]);
        }
    }
    f32x16 acc[VT];
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][e] = 0.0f;
    float m = NONE, l = 0.0f;
    bool far = false;
    const int krow = (lr & 0x13) | (lr >> 3 & 1) << 2 | (lr >> 2 & 1) << 3;       // key of score row lr: bits 2 and 3 changed over
    if (begin < end) {
        if (!whole(begin, page)) { asm volatile(""); clean(0); }
        expand_all(0);
        load(next);
    }
    // Two pages in LDS: while the scores of one are formed on the matrix cores, the vector pipe makes the next one f16; the products with the values run among the exponentials
    for (int i = begin, stage = 0; i < end; ++i, stage ^= 1) {
        const int after = page_of(i + 2), key0 = page_at(see, i) * PM_PAGE;
        const bool all = whole(i, page), there = page >= 0, dirty = i + 1 < end && !whole(i + 1, next);
        page = next; next = after;
        __syncthreads();                                   // (this page is there, the other stage and its flags are read)
        if (dirty) { asm volatile(""); clean(stage ^ 1); }
        const char * k_l = lds + stage * STAGE, * v_l = k_l + PM_PAGE * KL;
        f32x16 sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[t][e] = 0.0f;
        // a matrix instruction, its share of the vector work, and so on: in the order that stands here (the compiler would put the products together, which then wait for each other)
        auto key = [&](int q) __attribute__((always_inline)) { return *(const f16x8 *) (k_l + (q / KS * 32 + krow) * KL + (q % KS * 2 + hf) * 16); };
        f16x8 kf[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) kf[q] = key(q);
#pragma unroll
        for (int q = 0; q < 2 * KS; ++q) {
            const f16x8 k = kf[q % AHEAD];
            if (q + AHEAD < 2 * KS) kf[q % AHEAD] = key(q + AHEAD);
            sc[q / KS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[q % KS], sc[q / KS], 0, 0, 0);
            if (WIDE) sc[q / KS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[q % KS], sc[q / KS], 0, 0, 0);
            expand(q, stage ^ 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        load(next);
        if (!w_on || key0 > w_hi) continue;                // (a path of its own around the products too costs the registers of both)
        if (!all) {
            asm volatile("");
            const int last = there ? pos : -1;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t bad = *(const uint16_t *) (bad_l[stage] + t * 4 + hf * 2);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + t * 16 + 8 * hf + e;
                    const bool ok = key <= last && (key >= low || key < a.first);
                    sc[t >> 1][(t & 1) * 8 + e] = ok ? (bad >> ((e >> 2) * 8 + (e & 3)) & 1 ? NAN : sc[t >> 1][(t & 1) * 8 + e]) : -INFINITY;
                }
            }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[t][e]);
        mx = fmaxf(fmaxf(mx, __builtin_bit_cast(float, other_half(__builtin_bit_cast(uint32_t, mx)))) * cf, NONE);
        if (__any(mx > m + SLACK)) {
            const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= corr;
            far |= __any(fabsf(mn) > FAR && mn > NONE);
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] *= corr;
        }
        float k = cf, mo = HELD - m;
        if (far) {
            asm volatile("");
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[t][e] = sc[t][e] * k - m;
            k = 1.0f; mo = HELD;
        }
        f16x2 ph[2][4], pl[2][4];                          // probabilities of 16 keys, and of the next 16
        auto weigh = [&](int j, int e) __attribute__((always_inline)) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[j >> 1][(j & 1) * 8 + 2 * e], k, mo)), q = __builtin_amdgcn_exp2f(fmaf(sc[j >> 1][(j & 1) * 8 + 2 * e + 1], k, mo));
            l += p; l += q;
            const f16x2 h = {(_Float16) p, (_Float16) q};
            ph[j & 1][e] = h;
            if (WIDE) pl[j & 1][e] = f16x2{(_Float16) (p - (float) h.x), (_Float16) (q - (float) h.y)};
        };
        auto value = [&](int q) __attribute__((always_inline)) { return *(const f16x8 *) (v_l + (q % VT * 32 + lr) * VL + (q / VT * 2 + hf) * 16); };
        f16x8 vf[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) vf[q] = value(q);
#pragma unroll
        for (int e = 0; e < 4; ++e) weigh(0, e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < 4 * VT; ++q) {
            const int j = q / VT, t = q % VT;
            const f16x2 * h = ph[j & 1], * w = pl[j & 1];
            const f16x8 v = vf[q % AHEAD];
            if (q + AHEAD < 4 * VT) vf[q % AHEAD] = value(q + AHEAD);
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, eight(h[0], h[1], h[2], h[3]), acc[t], 0, 0, 0);
            if (WIDE) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, eight(w[0], w[1], w[2], w[3]), acc[t], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) if (j < 3 && e * VT / 4 == t) weigh(j + 1, e);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    l += __shfl_xor(l, 32);
    __syncthreads();
    if (splits == 1) {
        if (!on) return;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        T * o = (T *) a.out + (size_t) row * a.ldo + ch * D;
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int e = 0; e < 16; e += 4) st_out(o + t * 32 + 2 * e + 4 * hf, f32x4{acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]} * f);
        return;
    }
    float * part = a.work + slot * splits * TC * (D + 2);
    // (through LDS: a lane holds pieces of one column, memory wants whole lines)
    constexpr int LD = D + 4;
    float * sums = (float *) lds + wave * 32 * LD;
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(f32x4 *) (sums + lr * LD + t * 32 + 2 * e + 4 * hf) = f32x4{acc[t][e], acc[t][e + 1], acc[t][e + 2], acc[t][e + 3]};
    if (hf == 0 && col < cols) *(PM_G f32x2 *) (part + (size_t) splits * TC * D + (s * TC + col) * 2) = f32x2{m, l};
    __syncthreads();
    for (int o = threadIdx.x; o < cols * (D / 4); o += 256)
        *(PM_G f32x4 *) (part + (size_t) s * TC * D + o * 4) = *(const f32x4 *) ((const float *) lds + o / (D / 4) * LD + o % (D / 4) * 4);
}

// ---- joining split keys: partial sums per slot [splits][COLS][D], then [splits][COLS][maximum, sum]. A launch of its own: the workgroup of a slot that ends last could do it too, but it
// reads 2 MB (128 columns, 32 splits) alone, and waits for three trips to memory that other XCDs have written to; 64 tokens behind 30000 took 118 us that way ------------------------------
__host__ __device__ constexpr size_t join_factors(int splits, int each) { return ((size_t) splits * each * 8 + 15) & ~(size_t) 15; }      // bytes
template <typename T, int D, int COLS> __global__ __launch_bounds__(256) void join_kernel(pm_kv4_cache c, pm_kv4_attn a, int passes, int splits, int each) {
    extern __shared__ __attribute__((aligned(16))) char lds_j[];          // [splits][each][factor, sum], then the sums of groups of splits, at a multiple of 16 bytes
    __shared__ float inv[COLS];
    float * ml = (float *) lds_j, * sums = (float *) (lds_j + join_factors(splits, each));
    const int blocks = (COLS + each - 1) / each, first = blockIdx.x % blocks * each, G = c.G, R = a.H / G;
    const size_t slot = blockIdx.x / blocks;
    const int g = slot % G, pass = slot / G % passes;
    const int32_t * tile = uniform_const_ptr(a.tiles) + slot / G / passes * 4;
    const int row0 = tile[0], n = tile[1] < a.tile_tokens ? tile[1] : a.tile_tokens, room = COLS - first < each ? COLS - first : each, left = n * R - pass * COLS - first, cols = left < room ? left : room;
    if (n < 1 || cols < 1) return;
    const float * part = a.work + slot * splits * COLS * (D + 2) + first * D, * part_ml = a.work + slot * splits * COLS * (D + 2) + (size_t) splits * COLS * D + first * 2;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, items = cols * (D / 4), groups = items < 256 ? 256 / items : 1;
    // the first splits of this thread's column are on their way while the factors are formed
    constexpr int KB = 16;
    const int it0 = threadIdx.x % items, grp = groups > 1 ? threadIdx.x / items : 0;
    f32x4 r[KB];
    auto fetch = [&](int it, int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < KB; ++k) {
            const int z = k0 + k * groups < splits ? k0 + k * groups : splits - 1;
            r[k] = *(const PM_G f32x4 *) (part + ((size_t) z * COLS + it / (D / 4)) * D + it % (D / 4) * 4);
        }
    };
    fetch(it0, grp);
    for (int o = threadIdx.x; o < splits * cols; o += 256) {
        const f32x2 v = *(const PM_G f32x2 *) (part_ml + (o / cols * COLS + o % cols) * 2);
        ml[(o / cols * each + o % cols) * 2] = v.x; ml[(o / cols * each + o % cols) * 2 + 1] = v.y;
    }
    __syncthreads();
    for (int col = wave; col < cols; col += 4) {           // maximum and sum of a column by a wave; the factors of its splits take the place of their maxima
        float M = NONE, L = 0.0f;
        for (int k = lane; k < splits; k += 64) M = fmaxf(M, ml[(k * each + col) * 2]);
        M = all_max(M);
        for (int k = lane; k < splits; k += 64) { const float f = __builtin_amdgcn_exp2f(ml[(k * each + col) * 2] - M); ml[(k * each + col) * 2] = f; L = fmaf(ml[(k * each + col) * 2 + 1], f, L); }
        L = wave_sum(L);
        if (lane == 0) inv[col] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    __syncthreads();
    auto store = [&](int it, f32x4 v) __attribute__((always_inline)) {
        const int k = pass * COLS + first + it / (D / 4), row = row0 + k / R;
        if ((unsigned) row < (unsigned) a.n_tokens) st_out((T *) a.out + (size_t) row * a.ldo + (g * R + k % R) * D + it % (D / 4) * 4, v * inv[it / (D / 4)]);
    };
    for (int o = threadIdx.x; o < items * groups; o += 256) {
        const int it = o % items;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = grp; k0 < splits; k0 += KB * groups) {
            if (o != (int) threadIdx.x || k0 != grp) fetch(it, k0);
#pragma unroll
            for (int k = 0; k < KB; ++k)
                if (k0 + k * groups < splits) {
                    const float f = ml[((k0 + k * groups) * each + it / (D / 4)) * 2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(r[k][e], f, v[e]);
                }
        }
        if (groups == 1) store(it, v);
        else *(f32x4 *) (sums + o * 4) = v;
    }
    if (groups == 1) return;
    __syncthreads();
    for (int it = threadIdx.x; it < items; it += 256) {
        f32x4 v = *(const f32x4 *) (sums + it * 4);
        for (int k = 1; k < groups; ++k) v += *(const f32x4 *) (sums + (k * items + it) * 4);
        store(it, v);
    }
}

// FEW_WANT: one workgroup of 8 waves per CU is enough to fill the memory's queues, and every split costs its join. 32 tokens of 8 KV heads behind 8190 keys: 256 workgroups 67 us, 512 73, 1024 (of
// 4 waves) 80; one token behind 262100: 72, 72, 82. FEW_COLS: up to there rows of keys are read again per 32 columns; 8 x 16 tokens x 4 heads behind 4000 34 us, as one tile of 128 columns 38.
// FEW_PAGES: wider tiles go that way too where their workgroups are one round and all of them together read no more pages than this. 64, 128, 256 tokens of 32 + 8 heads of 128: behind 500 16, 19,
// 16 us, as tiles 23, 24, 28; behind 2000 (528, 1088, 2304 pages) 21, 26, 30 and 26, 29, 34; behind 4000 (1040, 2080, 4224 pages) 25, 34, 46 and 27, 31, 43. 512 tokens (512 workgroups) 26 us, as tiles
// 21. (No number of pages parts all of these: 256 tokens behind 2000 go the slower way, by 4 us.)
// FEW_JOIN: a join costs as much as FEW_JOIN / d + 2 pages of a workgroup, which the splits have to save. One token of 8 KV heads of 128 behind 500, 700, 1000, 1500: 9.0, 10.4, 11.7, 14.7 us in one,
// 11.4 .. 11.5 split; of 64: 7.4, 8.3, 9.2, 11.2 and 10.5 .. 10.8; of 256: 12.7, 15.1, 17.1, 21.4 and 13.7 .. 14.0.
// TILES_WANT: two workgroups per CU (one from heads of 192 on) share its matrix cores: 1.6 times the time of one, not 2. 512 tokens of 32 + 8 heads of 128 behind 12000 147 us, with 256 167. Partial sums
// are written and read, 2 * 128 (d + 2) floats per split, so splits have to save 3 pages and one more per 54 of them: 1000 tokens behind 300 42 us, in 2 splits 55; behind 12000 293 and 272; 320
// behind 900 34 in one, 28 in 6; 512 of 16 + 4 heads of 256 behind 4000 97 in 4, 81 in 2. LEAST: a step for every wave; a page's work for a join.
constexpr int FEW_WANT = 256, FEW_LEAST = 4, FEW_MOST = 128, FEW_COLS = 64, FEW_PAGES = 1536, FEW_JOIN = 1100, TILES_WANT = 512, TILES_LEAST = 4, TILES_MOST = 32;
// workgroups over which the keys of a slot are split: as many as fill the chip, none with less than `least` pages, and what the scratch holds
int splits_of(const pm_kv4_attn & a, int64_t pages, int64_t slots, int64_t busy, int want, int least, int most, int64_t floats) {
    const int64_t room = a.work ? (int64_t) a.work_floats / (slots * floats) : 1;
    int64_t n = want / busy;                               // (rounded up, the last ones are a second round: 6 tokens of 8 KV heads behind 8000 27 us instead of 22)
    n = n < pages / least ? n : pages / least;
    n = n < room ? n : room;
    n = n < most ? n : most;
    return n < 1 ? 1 : (int) n;
}
constexpr int columns_of(int nb, bool wide) { return nb <= (wide ? 3 : 4) ? 2 : 1; }       // tiles of 16 columns that a workgroup of few_kernel has registers for
pm_kv4_plan plan_of(int nb, bool wide, const pm_kv4_cache & c, const pm_kv4_attn & a) {
    const int R = a.H / c.G, D = nb * 32, CT = columns_of(nb, wide);
    const int64_t seen = (int64_t) a.window + a.tile_tokens + 128 + a.first, keys = a.window > 0 && seen < a.max_keys ? seen : a.max_keys, pages = (keys + PM_PAGE - 1) / PM_PAGE;
    // columns of a tile on the average: tile_tokens only bounds them
    const int64_t cols = (int64_t) R * (a.n_tokens / a.n_tiles < a.tile_tokens ? (a.n_tokens + a.n_tiles - 1) / a.n_tiles : a.tile_tokens), tiles = (int64_t) a.n_tiles * c.G;
    pm_kv4_plan p{};
    if (a.tile_tokens == 1 || cols <= FEW_COLS || (tiles * ((cols + 16 * CT - 1) / (16 * CT)) <= FEW_WANT && tiles * pages <= FEW_PAGES)) {
        const int ct = cols > 16 ? CT : 1;
        p.cols = 16 * ct;
        // (all passes side by side where that is one round and most of them have work: 40 tokens in tiles of 32 behind 100 11 us, with as many workgroups as the average wants 18)
        const int average = (int) ((cols + p.cols - 1) / p.cols);
        p.passes = (R * a.tile_tokens + p.cols - 1) / p.cols;
        p.launched = ct > 1 && (average * 2 <= p.passes || tiles * p.passes > FEW_WANT) ? average : p.passes;
        const int64_t slots = tiles * p.passes, busy = tiles * p.launched;
        p.splits = splits_of(a, pages, slots, busy, FEW_WANT, FEW_LEAST, FEW_MOST, p.cols * (D + 2));
        if ((pages - (pages + p.splits - 1) / p.splits - 2) * D < FEW_JOIN) p.splits = 1;
        p.groups = busy * p.splits;
        p.fits = p.groups < 1 << 23;                       // (a launch has fewer than 2^32 threads; that of the joins is small, as splits make one round at the most)
        return p;
    }
    p.cols = TC; p.passes = p.launched = 1;
    p.splits = splits_of(a, pages, tiles, tiles, nb <= 4 ? TILES_WANT : TILES_WANT / 2, TILES_LEAST, TILES_MOST, TC * (D + 2));
    if (pages - (tiles * p.splits > TILES_WANT / 2 ? 1.6 : 1.0) * (double) ((pages + p.splits - 1) / p.splits) < 3.0 + (double) (tiles * p.splits) / 54.0) p.splits = 1;
    p.groups = tiles * p.splits;
    p.fits = p.groups < 1 << 24;
    return p;
}

// columns per workgroup: the joined values of a thread come from about 16 splits
template <typename T, int D, int COLS> void join(const pm_kv4_cache & c, const pm_kv4_attn & a, const pm_kv4_plan & p, hipStream_t st) {
    const int most = 1024 / D, want = 16384 / (D * p.splits), each = want < 1 ? 1 : want < most ? want : most;
    const int64_t slots = (int64_t) a.n_tiles * c.G * p.passes;
    hipLaunchKernelGGL((join_kernel<T, D, COLS>), dim3((unsigned) (slots * ((COLS + each - 1) / each))), dim3(256), join_factors(p.splits, each) + 4096, st, c, a, p.passes, p.splits, each);
}
template <typename T, int NB, int CT> void few(const pm_kv4_cache & c, const pm_kv4_attn & a, const pm_kv4_plan & p, hipStream_t st) {
    constexpr int D = NB * 32;
    const auto kern = few_kernel<T, NB, sizeof(T) == 4, CT>;
    const size_t ring = (size_t) FW * STAGES * pm_step<NB>::BYTES, acc = (size_t) FW * 16 * (D + 4) * 4, lds = ring > acc ? ring : acc;
    pm_allow_big_lds((const void *) kern, lds);
    hipLaunchKernelGGL(kern, dim3((unsigned) p.groups), dim3(FW * 64), lds, st, c, a, p.launched, p.passes, p.splits);
    if (p.splits > 1) join<T, D, 16 * CT>(c, a, p, st);
}
template <typename T, int NB> int launch(const pm_kv4_cache & c, const pm_kv4_attn & a, hipStream_t st) {
    constexpr int D = NB * 32;
    constexpr bool WIDE = sizeof(T) == 4;
    const pm_kv4_plan p = plan_of(NB, WIDE, c, a);
    if (!p.fits) return PM355_E_SHAPE;
    if (p.cols != TC) {
        if constexpr (columns_of(NB, WIDE) == 2) if (p.cols == 32) { few<T, NB, 2>(c, a, p, st); return 0; }
        few<T, NB, 1>(c, a, p, st);
        return 0;
    }
    const size_t lds = 2 * ((size_t) PM_PAGE * (D * 2 + 16) + D * (PM_PAGE * 2 + 16));
    static_assert(2 * (PM_PAGE * (D * 2 + 16) + D * (PM_PAGE * 2 + 16)) >= TC * (D + 4) * 4, "the partial sums go through the pages' LDS");
    pm_allow_big_lds((const void *) tiles_kernel<T, NB, WIDE>, lds);
    hipLaunchKernelGGL((tiles_kernel<T, NB, WIDE>), dim3((unsigned) (a.n_tiles * (int64_t) c.G), p.splits), dim3(256), lds, st, c, a, p.splits);
    if (p.splits > 1) join<T, D, TC>(c, a, p, st);
    return 0;
}

} // namespace

// (slots * splits * columns is 128 times what prompts want at the most: few columns have 256 workgroups of up to 32, and up to four times as many slots as workgroups for them)
size_t pm_kv4_work_floats(int H, int G, int d) { return (size_t) (d <= 128 ? TILES_WANT : TILES_WANT / 2) * TC * (d + 2); }
pm_kv4_plan pm_attn_kv4_plan(const pm_kv4_cache & c, const pm_kv4_attn & a) { return plan_of(c.d / 32, a.type != PM_BF16, c, a); }
int pm_launch_attn_kv4(const pm_kv4_cache & c, const pm_kv4_attn & a, hipStream_t st) {
#define PM_CALL(NB) return a.type == PM_BF16 ? launch<uint16_t, NB>(c, a, st) : launch<float, NB>(c, a, st)
    switch (c.d) { case 64: PM_CALL(2); case 96: PM_CALL(3); case 128: PM_CALL(4); case 192: PM_CALL(6); case 256: PM_CALL(8); }
    return PM355_E_UNSUPPORTED;
}
