// attn_kv4.hip — attention over pages held in 4 bits: causal, with a sliding window and first tokens that stay visible.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp2(cf q k_j - max), over the j that the query sees; one pass over the keys with the running maximum and sum, both products on the f16 matrix cores.
// Keys and values become f16 in registers: a pair of codes is masked out of a word over the bits of 1024, less 1032, times the scale - 3.25 packed operations for two values (the words are
// ordered so that a mask gives a pair that an operand wants). Queries are brought to [1, 2) by a power of two per row, exact for bf16; WIDE (32-bit rows) holds queries and probabilities as
// pairs of f16 and makes two products of each. Probabilities are held times 2^8, so that f16 has its steps of 2^-11 down to p = 2^-22.
// S^T = K Q^T is computed with the key rows permuted so that a lane's score registers are its P operand of O^T = V^T P^T.
//   few    up to 16 columns (tokens x query heads of a KV head) per workgroup, 32 keys per wave and step straight from memory, keys split over waves and workgroups: bound by memory
//   tiles  128 columns per workgroup, a page at a time through LDS, where it is made f16 once for all four waves: bound by the matrix cores and the vector work on scores
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include "../../include/prima_mi355.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -1e30f;                             // running maximum before the first visible key
constexpr float HELD = 8.0f;                               // probabilities are held times 2^HELD
constexpr int TICKETS = 65536;                             // words of the scratch in front of the partial sums

// N words (N halves) that lie side by side, a multiple of 4 N (2 N) bytes into a slab
template <int N> __device__ __forceinline__ void ld_words(const char * p, uint32_t * w) {
    if constexpr (N == 1) w[0] = *(const PM_G uint32_t *) p;
    else if constexpr (N == 2) { const u32x2 t = *(const PM_G u32x2 *) p; w[0] = t.x; w[1] = t.y; }
    else if constexpr (N == 3) { const u32x3 t = *(const PM_G u32x3 *) p; w[0] = t.x; w[1] = t.y; w[2] = t.z; }
    else if constexpr (N == 4) { const u32x4 t = *(const PM_G u32x4 *) p; w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
    else { ld_words<N / 2>(p, w); ld_words<N / 2>(p + 2 * N, w + N / 2); }
}
template <int N> __device__ __forceinline__ void ld_halves(const char * p, uint32_t * w) {
    if constexpr (N == 3) {
        const PM_G uint16_t * h = (const PM_G uint16_t *) p;
        w[0] = h[0] | (uint32_t) h[1] << 16; w[1] = h[2];
    } else ld_words<N / 2>(p, w);
}
__device__ __forceinline__ f16x2 half_of(const uint32_t * w, int i) {      // value i of packed halves, twice
    const uint32_t h = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffff;
    return __builtin_bit_cast(f16x2, h | h << 16);
}
// the codes at nibble p of both halves of a word, times scales: two f16 values
__device__ __forceinline__ f16x2 pair(uint32_t w, int p, f16x2 s) {
    const f16x2 n = __builtin_bit_cast(f16x2, (w >> (4 * p) & 0x000f000fu) | 0x64006400u);
    return (n - f16x2{(_Float16) 1032.0f, (_Float16) 1032.0f}) * s;
}
__device__ __forceinline__ f16x8 eight(f16x2 a, f16x2 b, f16x2 c, f16x2 d) { return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; }
// scales beyond what the cache store makes (8188: its codes stay finite), NaN and infinities become 0; bits 0, 1: which
__device__ __forceinline__ uint32_t finite(uint32_t & s) {
    const uint32_t lo = (s & 0x7fffu) > 0x6fffu, hi = (s & 0x7fffffffu) > 0x6fffffffu;
    s &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    return lo | hi << 1;
}
__device__ __forceinline__ void st_shared(float * p, float v) { __hip_atomic_store((PM_G float *) p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float ld_shared(const float * p) { return __hip_atomic_load((const PM_G float *) p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

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
// 2^-e with the sign of scale for a row whose largest magnitude is in [2^e, 2^(e + 1)); cf = |scale| log2(e) 2^e
__device__ __forceinline__ float row_factor(float most, float scale, float & cf) {
    int e = (int) (__builtin_bit_cast(uint32_t, most) >> 23 & 255) - 127;
    e = e < -100 ? -100 : e > 100 ? 0 : e;                 // (a row of zeros; rows that are not finite stay so)
    cf = fmaxf(fabsf(scale) * LOG2E * ldexpf(1.0f, e), 1e-30f);
    return copysignf(ldexpf(1.0f, -e), scale);
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
constexpr int FW = 4;                                      // waves of a workgroup
template <int NB> struct pm_chunk { uint32_t k[2][NB], ks[2][(NB + 1) / 2], v[2][NB], vs[NB][4]; };      // codes and scales of 32 keys as a lane wants them

template <typename T, int NB, bool WIDE> __global__ __launch_bounds__(FW * 64) void few_kernel(pm_kv4_cache c, pm_kv4_attn a, int splits) {
    constexpr int D = NB * 32, VT = D / 16, LD = D + 4;
    typedef pm_kv4_slab<NB> S;
    extern __shared__ __attribute__((aligned(16))) float acc_l[];         // [FW][16][LD]
    __shared__ float m_l[FW][16], l_l[FW][16], ml[64 * 32];
    __shared__ int is_last;
    const int G = c.G, R = a.H / G, HT = (R + 15) / 16, gh = blockIdx.x % (G * HT), g = gh / HT, ht = gh % HT, s = blockIdx.y;
    const size_t slot = blockIdx.x;
    const int32_t * tile = uniform_const_ptr(a.tiles) + blockIdx.x / (G * HT) * 4;
    const int row0 = tile[0], seq = tile[3], pos0 = tile[2] < 0x7fffff00 ? tile[2] : 0x7fffff00, n = tile[1] < a.tile_tokens ? tile[1] : a.tile_tokens;
    if (n < 1) return;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    const int nh = R <= 16 ? R : R - ht * 16 < 16 ? R - ht * 16 : 16, cols = n * nh;
    const int ct = lr < cols ? lr / nh : 0, ch = g * R + ht * 16 + (lr < cols ? lr % nh : 0);             // token and head of this lane's column
    const pm_seen see = seen_by(c, a, pos0, n);
    const int pos = lr < cols && pos0 >= 0 ? pos0 + ct : -1, low = a.window > 0 ? pos - a.window + 1 : 0;
    const int per = (see.count + splits - 1) / splits, end = 2 * ((s + 1) * per < see.count ? (s + 1) * per : see.count);
    const int32_t * table = uniform_const_ptr(c.table) + (size_t) ((unsigned) seq < (unsigned) c.n_seq ? seq : 0) * c.table_ld;
    const bool known = (unsigned) seq < (unsigned) c.n_seq;
    const char * head = c.pages + (size_t) g * S::BYTES;
    auto page_of = [&](int i) __attribute__((always_inline)) { if (!known || i >= end) return -1; const int p = table[page_at(see, i >> 1)]; return (unsigned) p < (unsigned) c.n_pages ? p : -1; };
    const int krow = 8 * (lr >> 2) + (lr & 3);             // key of score row lr in the first 16 of a step (the second: + 4)
    auto load = [&](pm_chunk<NB> & x, int i, int page) __attribute__((always_inline)) {
        if (page < 0) return;
        const char * slab = head + (size_t) page * G * S::BYTES;
        const int key = (i & 1) * 32;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            ld_words<NB>(slab + S::K + (key + krow + 4 * b) * 16 * NB + lg * 4 * NB, x.k[b]);
            ld_words<NB>(slab + S::V + ((key >> 2) + 2 * lg + b) * 64 * NB + lr * 4 * NB, x.v[b]);
            ld_halves<NB>(slab + S::KS + (key + krow + 4 * b) * 2 * NB, x.ks[b]);
        }
#pragma unroll
        for (int w = 0; w < NB; ++w) ld_words<4>(slab + S::VS + (w * PM_PAGE + key + 8 * lg) * 2, x.vs[w]);
    };
    int i = 2 * s * per + wave, page = page_of(i), next = page_of(i + FW);
    pm_chunk<NB> x0, x1;
    load(x0, i, page);

    f16x8 qh[NB], ql[NB];
    float cf;
    {
        const int row = row0 + ct;
        const bool on = lr < cols && (unsigned) row < (unsigned) a.n_tokens;
        float x[NB][8], most = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
            if (on) ld_query<T>((const T *) a.q + (size_t) row * a.ldq + ch * D + b * 32 + lg * 8, x[b]);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[b][j]));
        }
        most = fmaxf(most, __shfl_xor(most, 16)); most = fmaxf(most, __shfl_xor(most, 32));
        const float f = row_factor(most, a.scale, cf);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] *= f;
            split_f16(x[b], qh[b], ql[b]);
        }
    }
    f32x4 acc[VT];
#pragma unroll
    for (int t = 0; t < VT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = NONE, l = 0.0f;
    auto step = [&](pm_chunk<NB> & x, int i) __attribute__((always_inline)) {
        const int key0 = page_at(see, i >> 1) * PM_PAGE + (i & 1) * 32 + lg * 8;      // the lane's eight keys
        f32x4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const f16x2 sa = half_of(x.ks[0], b), sb = half_of(x.ks[1], b);
            const f16x8 ka = eight(pair(x.k[0][b], 0, sa), pair(x.k[0][b], 1, sa), pair(x.k[0][b], 2, sa), pair(x.k[0][b], 3, sa));
            const f16x8 kb = eight(pair(x.k[1][b], 0, sb), pair(x.k[1][b], 1, sb), pair(x.k[1][b], 2, sb), pair(x.k[1][b], 3, sb));
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[b], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qh[b], s1, 0, 0, 0);
            if (WIDE) { s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[b], s0, 0, 0, 0); s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, ql[b], s1, 0, 0, 0); }
        }
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = j < 4 ? s0[j & 3] : s1[j & 3];
        // a step that not every column sees whole: hidden keys count nothing, whatever their slots hold
        const int k0 = key0 - lg * 8;
        if (k0 + 31 > see.lo || (a.window > 0 && k0 <= see.hi - a.window)) {
            uint32_t bad = 0;
#pragma unroll
            for (int w = 0; w < NB; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) bad |= finite(x.vs[w][j]) << 2 * j;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + j;
                const bool ok = key <= pos && (key >= low || key < a.first);
                f[j] = ok ? (bad >> j & 1 ? NAN : f[j]) : -INFINITY;
            }
        }
        float mx = f[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, f[j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16)); mx = fmaxf(mx, __shfl_xor(mx, 32));
        mx = fmaxf(mx * cf, NONE);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= corr;
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] *= corr;
        }
        f16x8 ph, pl;
        const float mo = HELD - m;
#pragma unroll
        for (int j = 0; j < 8; ++j) { f[j] = __builtin_amdgcn_exp2f(fmaf(f[j], cf, mo)); l += f[j]; }
        split_f16(f, ph, pl);
#pragma unroll
        for (int w = 0; w < NB; ++w) {
            f16x2 sc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[j] = __builtin_bit_cast(f16x2, x.vs[w][j]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f16x8 v = eight(pair(x.v[0][w], h, sc[0]), pair(x.v[0][w], h + 2, sc[1]), pair(x.v[1][w], h, sc[2]), pair(x.v[1][w], h + 2, sc[3]));
                acc[2 * w + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, acc[2 * w + h], 0, 0, 0);
                if (WIDE) acc[2 * w + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, acc[2 * w + h], 0, 0, 0);
            }
        }
    };
    // the next 32 keys are on their way while these are worked on, and the page after them is looked up
    for (; i < end; i += 2 * FW) {
        const int after = page_of(i + 2 * FW), then = page_of(i + 3 * FW);
        load(x1, i + FW, next);
        if (page >= 0) step(x0, i);
        load(x0, i + 2 * FW, after);
        if (next >= 0) step(x1, i + FW);
        page = after; next = then;
    }
    l += __shfl_xor(l, 16); l += __shfl_xor(l, 32);
    if (lr < cols) {
#pragma unroll
        for (int t = 0; t < VT; ++t) *(f32x4 *) (acc_l + (wave * 16 + lr) * LD + t * 16 + lg * 4) = acc[t];
        if (lg == 0) { m_l[wave][lr] = m; l_l[wave][lr] = l; }
    }
    __syncthreads();
    auto store = [&](int col, int d, float o) {
        const int row = row0 + col / nh;
        if ((unsigned) row < (unsigned) a.n_tokens) ((T *) a.out)[(size_t) row * a.ldo + (g * R + ht * 16 + col % nh) * D + d] = from_f<T>(o);
    };
    float * part = a.work + TICKETS + slot * splits * 16 * (D + 2);
    for (int o = threadIdx.x; o < cols * D; o += FW * 64) {
        const int col = o / D, d = o % D;
        float M = NONE, v = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < FW; ++w) M = fmaxf(M, m_l[w][col]);
#pragma unroll
        for (int w = 0; w < FW; ++w) { const float f = __builtin_amdgcn_exp2f(m_l[w][col] - M); v += acc_l[(w * 16 + col) * LD + d] * f; sum += l_l[w][col] * f; }
        if (splits == 1) store(col, d, sum == 0.0f ? 0.0f : v / sum);
        else {
            float * r = part + (s * 16 + col) * (D + 2);
            st_shared(r + d, v);
            if (d == 0) { st_shared(r + D, M); st_shared(r + D + 1, sum); }
        }
    }
    if (splits == 1) return;
    // partial sums out, then a ticket; the workgroup that draws the last one joins them in their order and leaves the ticket as it was
    pm_vm_drain();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned * tk = (unsigned *) a.work + slot;
        is_last = __hip_atomic_fetch_add(tk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned) splits - 1;
        if (is_last) __hip_atomic_store(tk, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!is_last) return;
    for (int o = threadIdx.x; o < splits * 32; o += FW * 64) if ((o >> 1 & 15) < cols) ml[o] = ld_shared(part + (o >> 1) * (D + 2) + D + (o & 1));
    __syncthreads();
    for (int o = threadIdx.x; o < cols * D; o += FW * 64) {
        const int col = o / D, d = o % D;
        float M = NONE, v = 0.0f, sum = 0.0f;
        for (int k = 0; k < splits; ++k) M = fmaxf(M, ml[(k * 16 + col) * 2]);
        for (int k0 = 0; k0 < splits; k0 += 8) {
            float r[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = ld_shared(part + ((k0 + k < splits ? k0 + k : splits - 1) * 16 + col) * (D + 2) + d);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k < splits) { const float f = __builtin_amdgcn_exp2f(ml[((k0 + k) * 16 + col) * 2] - M); v += r[k] * f; sum += ml[((k0 + k) * 16 + col) * 2 + 1] * f; }
        }
        store(col, d, sum == 0.0f ? 0.0f : v / sum);
    }
}

// ---- prompts ----------------------------------------------------------------------------------------------------------------
constexpr int TC = 128;                                    // columns of a tile: 32 per wave

template <typename T, int NB, bool WIDE> __global__ __launch_bounds__(256) void tiles_kernel(pm_kv4_cache c, pm_kv4_attn a, int splits) {
    constexpr int D = NB * 32, KS = D / 16, VT = D / 32, KL = D * 2 + 16, VL = PM_PAGE * 2 + 16;      // LDS rows are an odd number of 16-byte pieces: no bank is asked twice
    typedef pm_kv4_slab<NB> S;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // K [64][KL], V^T [D][VL]
    char * k_l = lds, * v_l = lds + PM_PAGE * KL;
    __shared__ uint8_t bad_l[16];
    __shared__ int is_last;
    const int G = c.G, R = a.H / G, g = blockIdx.x % G, s = blockIdx.y;
    const int at = a.n_tiles - 1 - (int) (blockIdx.x / G);                // (later tiles see more keys: they start first)
    const size_t slot = blockIdx.x;
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
    uint32_t xk[NB], xks[(NB + 1) / 2], xv[NB], xvs[NB][2];
    auto load = [&](int page) __attribute__((always_inline)) {
        if (page < 0) return;
        const char * slab = head + (size_t) page * G * S::BYTES;
        ld_words<NB>(slab + S::K + kr * 16 * NB + kg * 4 * NB, xk);
        ld_halves<NB>(slab + S::KS + kr * 2 * NB, xks);
        ld_words<NB>(slab + S::V + vq * 64 * NB + vn * 4 * NB, xv);
#pragma unroll
        for (int w = 0; w < NB; ++w) ld_words<2>(slab + S::VS + (w * PM_PAGE + vq * 4) * 2, xvs[w]);
    };
    int page = page_of(begin);
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
    const int krow = (lr & 0x13) | (lr >> 3 & 1) << 2 | (lr >> 2 & 1) << 3;       // key of score row lr: bits 2 and 3 changed over
    for (int i = begin; i < end; ++i) {
        const int next = page_of(i + 1), key0 = page_at(see, i) * PM_PAGE;
        const bool whole = key0 + PM_PAGE - 1 <= see.lo && !(a.window > 0 && key0 <= see.hi - a.window);      // every column sees the page whole
        if (page >= 0) {
            __syncthreads();                               // (the page before is read)
            if (!whole) {
                uint32_t bad = 0;
#pragma unroll
                for (int w = 0; w < NB; ++w) bad |= finite(xvs[w][0]) | finite(xvs[w][1]) << 2;
                if (vn == 0) bad_l[vq] = (uint8_t) bad;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f16x2 sc = half_of(xks, b);
                *(f16x8 *) (k_l + kr * KL + (b * 4 + kg) * 16) = eight(pair(xk[b], 0, sc), pair(xk[b], 1, sc), pair(xk[b], 2, sc), pair(xk[b], 3, sc));
                const f16x2 s0 = __builtin_bit_cast(f16x2, xvs[b][0]), s1 = __builtin_bit_cast(f16x2, xvs[b][1]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *(u32x2 *) (v_l + (b * 32 + h * 16 + vn) * VL + vq * 8) = u32x2{__builtin_bit_cast(uint32_t, pair(xv[b], h, s0)), __builtin_bit_cast(uint32_t, pair(xv[b], h + 2, s1))};
            }
            __syncthreads();
        }
        load(next);
        const bool go = page >= 0 && w_on && key0 <= w_hi;
        page = next;
        if (!go) continue;
        f32x16 sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[t][e] = 0.0f;
#pragma unroll
            for (int b = 0; b < KS; ++b) {
                const f16x8 k = *(const f16x8 *) (k_l + (t * 32 + krow) * KL + (b * 2 + hf) * 16);
                sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[b], sc[t], 0, 0, 0);
                if (WIDE) sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[b], sc[t], 0, 0, 0);
            }
        }
        if (!whole)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int kk = t * 32 + 16 * (e >> 3) + 8 * hf + (e & 7), key = key0 + kk;
                    const bool ok = key <= pos && (key >= low || key < a.first);
                    sc[t][e] = ok ? (bad_l[kk >> 2] >> (kk & 3) & 1 ? NAN : sc[t][e]) : -INFINITY;
                }
        float mx = sc[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[t][e]);
        mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32)) * cf, NONE);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= corr;
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] *= corr;
        }
        const float mo = HELD - m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float p[8];
            f16x8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; ++e) { p[e] = __builtin_amdgcn_exp2f(fmaf(sc[j >> 1][(j & 1) * 8 + e], cf, mo)); l += p[e]; }
            split_f16(p, ph, pl);
#pragma unroll
            for (int t = 0; t < VT; ++t) {
                const f16x8 v = *(const f16x8 *) (v_l + (t * 32 + lr) * VL + (j * 2 + hf) * 16);
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, acc[t], 0, 0, 0);
                if (WIDE) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, acc[t], 0, 0, 0);
            }
        }
    }
    l += __shfl_xor(l, 32);
    if (splits == 1) {
        if (!on) return;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        T * o = (T *) a.out + (size_t) row * a.ldo + ch * D;
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = t * 32 + 2 * e + 4 * hf;
                if constexpr (sizeof(T) == 2) *(PM_G u16x4 *) (o + d) = u16x4{f2bf(acc[t][e] * f), f2bf(acc[t][e + 1] * f), f2bf(acc[t][e + 2] * f), f2bf(acc[t][e + 3] * f)};
                else *(PM_G f32x4 *) (o + d) = f32x4{acc[t][e] * f, acc[t][e + 1] * f, acc[t][e + 2] * f, acc[t][e + 3] * f};
            }
        return;
    }
    float * part = a.work + TICKETS + slot * splits * TC * (D + 2);
    if (col < cols) {
        float * r = part + ((size_t) s * TC + col) * (D + 2);
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) st_shared(r + t * 32 + 8 * (e >> 2) + 4 * hf + (e & 3), acc[t][e]);
        if (hf == 0) { st_shared(r + D, m); st_shared(r + D + 1, l); }
    }
    pm_vm_drain();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned * tk = (unsigned *) a.work + slot;
        is_last = __hip_atomic_fetch_add(tk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned) splits - 1;
        if (is_last) __hip_atomic_store(tk, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!is_last) return;
    for (int o = threadIdx.x; o < cols * D; o += 256) {
        const int k = o / D, d = o % D, to = row0 + k / R;
        const float * r = part + (size_t) k * (D + 2);
        float M = NONE, v = 0.0f, sum = 0.0f;
        for (int z = 0; z < splits; ++z) M = fmaxf(M, ld_shared(r + (size_t) z * TC * (D + 2) + D));
        for (int z = 0; z < splits; ++z) {
            const float * q = r + (size_t) z * TC * (D + 2);
            const float f = __builtin_amdgcn_exp2f(ld_shared(q + D) - M);
            v += ld_shared(q + d) * f; sum += ld_shared(q + D + 1) * f;
        }
        if ((unsigned) to < (unsigned) a.n_tokens) ((T *) a.out)[(size_t) to * a.ldo + (g * R + k % R) * D + d] = from_f<T>(sum == 0.0f ? 0.0f : v / sum);
    }
}

// workgroups over which the keys of a slot are split: as many as fill the chip, none with less than `least` pages, and what the scratch holds
int splits_of(const pm_kv4_attn & a, int64_t slots, int want, int least, int64_t floats) {
    const int64_t pages = ((int64_t) a.max_keys + PM_PAGE - 1) / PM_PAGE, room = a.work && a.work_floats > TICKETS ? (int64_t) (a.work_floats - TICKETS) / (slots * floats) : 1;
    int64_t n = (want + slots - 1) / slots;
    n = n < pages / least ? n : pages / least;
    n = n < room ? n : room;
    n = n < 64 ? n : 64;
    return slots > TICKETS || n < 1 ? 1 : (int) n;
}
constexpr int FEW_WANT = 1024, FEW_LEAST = 4, TILES_WANT = 512, TILES_LEAST = 8;

template <typename T, int NB> int launch(const pm_kv4_cache & c, pm_kv4_attn a, hipStream_t st) {
    constexpr int D = NB * 32;
    constexpr bool WIDE = sizeof(T) == 4;
    const int R = a.H / c.G;
    if (a.window > 0) { const int64_t most = (int64_t) a.window + a.tile_tokens + 128 + a.first; if (most < a.max_keys) a.max_keys = (int) most; }
    if (a.tile_tokens == 1 || R * a.tile_tokens <= 16) {
        const int64_t slots = (int64_t) a.n_tiles * c.G * ((R + 15) / 16);
        const size_t lds = (size_t) FW * 16 * (D + 4) * 4;
        const int splits = splits_of(a, slots, FEW_WANT, FEW_LEAST, 16 * (D + 2));
        pm_allow_big_lds((const void *) few_kernel<T, NB, WIDE>, lds);
        hipLaunchKernelGGL((few_kernel<T, NB, WIDE>), dim3((unsigned) slots, splits), dim3(FW * 64), lds, st, c, a, splits);
        return 0;
    }
    const int64_t slots = (int64_t) a.n_tiles * c.G;
    const size_t lds = (size_t) PM_PAGE * (D * 2 + 16) + D * (PM_PAGE * 2 + 16);
    const int splits = splits_of(a, slots, TILES_WANT, TILES_LEAST, TC * (D + 2));
    pm_allow_big_lds((const void *) tiles_kernel<T, NB, WIDE>, lds);
    hipLaunchKernelGGL((tiles_kernel<T, NB, WIDE>), dim3((unsigned) slots, splits), dim3(256), lds, st, c, a, splits);
    return 0;
}

} // namespace

// (slots * splits < want + slots, and slots < want where there are splits)
size_t pm_kv4_work_floats(int H, int G, int d) { return TICKETS + (size_t) 2 * TILES_WANT * TC * (d + 2); }
int pm_launch_attn_kv4(const pm_kv4_cache & c, const pm_kv4_attn & a, hipStream_t st) {
#define PM_CALL(NB) return a.type == PM_BF16 ? launch<uint16_t, NB>(c, a, st) : launch<float, NB>(c, a, st)
    switch (c.d) { case 64: PM_CALL(2); case 96: PM_CALL(3); case 128: PM_CALL(4); case 192: PM_CALL(6); case 256: PM_CALL(8); }
    return PM355_E_UNSUPPORTED;
}
