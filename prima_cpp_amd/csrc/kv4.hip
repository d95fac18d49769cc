// kv4.hip — into a 4-bit KV cache and out of it: per-head norm of queries and keys, rotation, rounding to 4 bits, one pass over the projections.
//
// y = x / sqrt(mean(x^2) + eps) w;  (a, b) -> (a cos - b sin, b cos + a sin) mscale at 2 pi frac(pos turns_i);  scale = f16(M / -8), code = clamp(rint(y / scale), -8, 7) + 8.
// Bound by memory: a row of (H + 2 G) d values is read once, H d values and 1.125 G d bytes are written. 6001 tokens of 32 + 8 heads of 128 (bf16, norm, rotation) 36 us for 130 MB, without keys and
// values 24 for 98 MB (the scattered bytes of the values are 4 us of the difference); 48 tokens of 64 + 8 heads 5.2 us, one token 4.0. Reading 6001 tokens back 9.7 us (31 MB).
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include "../../include/prima_mi355.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void st4(float * p, const float * v) { *(PM_G f32x4 *) p = f32x4{v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void st4(uint16_t * p, const float * v) { *(PM_G u16x4 *) p = u16x4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])}; }

// what the other lanes of a group of 2, 4, 8, 16, 32 hold, once the smaller groups agree: DPP within rows of 16, a lane swap between them
template <int M> __device__ __forceinline__ uint32_t other(uint32_t v) {
    if constexpr (M == 16) return other_row(v);
    else return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, M == 1 ? 0xB1 : M == 2 ? 0x4E : M == 4 ? 0x141 : 0x140, 0xF, 0xF, true);
}
template <int M> __device__ __forceinline__ float other(float v) { return __builtin_bit_cast(float, other<M>(__builtin_bit_cast(uint32_t, v))); }
template <int M> __device__ __forceinline__ double other(double v) {
    const u32x2 t = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{other<M>((uint32_t) t.x), other<M>((uint32_t) t.y)});
}
template <int LPH, typename F> __device__ __forceinline__ F head_sum(F v) {       // over the LPH lanes of a head row
    v += other<1>(v); v += other<2>(v); v += other<4>(v);
    if constexpr (LPH >= 16) v += other<8>(v);
    if constexpr (LPH >= 32) v += other<16>(v);
    return v;
}
// scale (f16 bits) of a block whose 32 values lie in four neighbouring lanes, 8 each; NaN where the row holds a NaN or an infinity
template <int LPH> __device__ __forceinline__ uint16_t block_scale(const float * x) {
    float hi = x[0], lo = x[0], bad = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { hi = fmaxf(hi, x[j]); lo = fminf(lo, x[j]); bad = fmaf(x[j], 0.0f, bad); }       // (0 * NaN, 0 * inf: NaN)
    hi = fmaxf(hi, other<1>(hi)); lo = fminf(lo, other<1>(lo));
    hi = fmaxf(hi, other<2>(hi)); lo = fminf(lo, other<2>(lo));
    bad = head_sum<LPH>(bad);
    const float s = fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -8188.0f), 8188.0f);
    return bad == 0.0f ? f2h(s) : (uint16_t) 0x7e00;
}
// codes 0 .. 15 of eight values. r = 1 / s to half a unit; x r, corrected by its remainder, is then x / s as rounded once, so that a tie between two codes is seen as one
__device__ __forceinline__ void block_codes(const float * x, uint16_t scale, float * c) {
    const float s = h2f(scale), r = s != 0.0f && s == s ? 1.0f / s : 0.0f;        // (an empty block, a row that is not finite)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = x[j] * r;
        c[j] = __builtin_amdgcn_fmed3f(rintf(fmaf(fmaf(-q, s, x[j]), r, q)), -8.0f, 7.0f) + 8.0f;
    }
}

// values of a lane on their way: two groups of four
template <typename T> struct pm_raw;
template <> struct pm_raw<float> { f32x4 a, b; };
template <> struct pm_raw<uint16_t> { u16x4 a, b; };
__device__ __forceinline__ void widen(const pm_raw<float> & r, float * v) { for (int j = 0; j < 4; ++j) { v[j] = r.a[j]; v[j + 4] = r.b[j]; } }
__device__ __forceinline__ void widen(const pm_raw<uint16_t> & r, float * v) { for (int j = 0; j < 4; ++j) { v[j] = bf2f(r.a[j]); v[j + 4] = bf2f(r.b[j]); } }
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); __builtin_amdgcn_wave_barrier(); }

// A wave takes 64 / LPH head rows at a time, 8 values per lane as two groups of 4: for pairs (i, i + n_rot / 2) the groups are the two halves of four pairs, otherwise they are neighbours;
// values of the cache are grouped as their bytes are, dimensions n and n + 16 of a block. LPH = 8, 16, 32: the smallest power of two that covers d / 8. A token belongs to one wave where
// there are many (the next rows are on their way while these are worked on, nothing is waited for but memory, and a quad's value bytes leave one workgroup), or to `parts` waves.
template <typename T, int NB> __global__ __launch_bounds__(256) void append_kernel(pm_kv4_cache c, pm_kv4_append a, int parts) {
    constexpr int D = NB * 32, LPH = NB <= 2 ? 8 : NB <= 4 ? 16 : 32, RPW = 64 / LPH;
    typedef pm_kv4_slab<NB> S;
    __shared__ double cs_l[4][PM_KV4_MAX_D / 2][2];
    __shared__ __attribute__((aligned(16))) float keys_l[4][RPW][D];
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane % LPH, sub = lane / LPH;
    const int t = (int) ((blockIdx.x * 4u + wave) / (unsigned) parts), part = (int) ((blockIdx.x * 4u + wave) % (unsigned) parts);
    if (t >= a.T) return;
    const int G = c.G, NG = (G + RPW - 1) / RPW, N = 2 * NG + (a.H + RPW - 1) / RPW, rot = a.turns ? a.n_rot : 0;
    const bool on = i * 8 < D, turn = i * 8 < rot;
    const int o0 = !on ? 0 : a.neox && turn ? i * 4 : i * 8, o1 = !on ? 4 : a.neox && turn ? i * 4 + rot / 2 : i * 8 + 4, ov = on ? (i >> 2) * 32 + (i & 3) * 4 : 0;
    const T * row = (const T *) a.proj + (size_t) t * a.ldp;
    // rows [0, NG): keys, [NG, 2 NG): values, then queries (no branch around the loads: rows that are not there are read as the last one)
    auto load = [&](int n) __attribute__((always_inline)) {
        const bool key = n < NG, val = !key && n < 2 * NG;
        int h = (key ? n : val ? n - NG : n - 2 * NG) * RPW + sub;
        const int most = key || val ? G : a.H;
        h = h < most ? h : most - 1;
        const T * p = row + ((key ? a.H : val ? a.H + G : 0) + h) * D;
        pm_raw<T> r;
        r.a = *(const PM_G decltype(r.a) *) (p + (val ? ov : o0));
        r.b = *(const PM_G decltype(r.a) *) (p + (val ? ov + 16 : o1));
        return r;
    };
    pm_raw<T> next = load(part);
    const int at = a.pos[t], pos = at < 0 ? 0 : at, page = pm_kv4_page(c, a.seq[t], at), slot = pos % PM_PAGE;
    char * const slab0 = c.pages + (size_t) (page < 0 ? 0 : page) * G * S::BYTES;
    double (*cs)[2] = cs_l[wave];
    for (int j = lane; j < rot / 2; j += 64) {
        const double u = (double) pos * a.turns[j];
        double s, k;
        sincospi(2.0 * (u - floor(u)), &s, &k);
        cs[j][0] = k * (double) a.mscale;
        cs[j][1] = s * (double) a.mscale;
    }
    lds_done();
    int n = part;
    float x[8];
    auto take = [&](int heads, int h) __attribute__((always_inline)) {       // this step's values, the next one's on their way; whether this lane has any
        widen(next, x);
        next = load(n + parts < N ? n + parts : n);
        const bool live = on && h < heads;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = live ? x[j] : 0.0f;
        return live;
    };
    // keys: 64 bits up to the one rounding to 32, so that a code never depends on the order of a sum
    for (; n < NG; n += parts) {
        const int h = n * RPW + sub;
        const bool live = take(G, h);
        double y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[j];
        if (a.norm) {
            double ss = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fma(y[j], y[j], ss);
            const double r = 1.0 / sqrt(head_sum<LPH>(ss) / D + (double) a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= r * (a.wk ? (double) a.wk[(j < 4 ? o0 : o1 - 4) + j] : 1.0);
        }
        if (turn)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                double & p = a.neox ? y[j] : y[2 * j], & q = a.neox ? y[j + 4] : y[2 * j + 1];
                const double k = cs[i * 4 + j][0], s = cs[i * 4 + j][1], u = p, v = q;
                p = u * k - v * s; q = v * k + u * s;
            }
        // into the order of the page: lane i holds dimensions 8 i .. 8 i + 7
        float * kb = keys_l[wave][sub];
        if (on)
#pragma unroll
            for (int j = 0; j < 4; ++j) { kb[o0 + j] = (float) y[j]; kb[o1 + j] = (float) y[j + 4]; }
        lds_done();
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = live ? kb[i * 8 + j] : 0.0f;
        lds_done();
        const uint16_t sb = block_scale<LPH>(x);
        float q[8];
        block_codes(x, sb, q);
        if (!live || page < 0) continue;
        char * slab = slab0 + (size_t) h * S::BYTES;
        // dimensions 0, 2, 4, 6 are the nibbles of the low half, 1, 3, 5, 7 of the high one
        const uint32_t lo = (uint32_t) fmaf(q[6], 4096.0f, fmaf(q[4], 256.0f, fmaf(q[2], 16.0f, q[0]))), hi = (uint32_t) fmaf(q[7], 4096.0f, fmaf(q[5], 256.0f, fmaf(q[3], 16.0f, q[1])));
        *(PM_G uint32_t *) (slab + S::K + slot * 16 * NB + (i & 3) * 4 * NB + (i >> 2) * 4) = lo | hi << 16;
        if ((i & 3) == 0) *(PM_G uint16_t *) (slab + S::KS + (slot * NB + (i >> 2)) * 2) = sb;
    }
    for (; n < 2 * NG; n += parts) {
        const int h = (n - NG) * RPW + sub;
        const bool live = take(G, h);
        const uint16_t sb = block_scale<LPH>(x);
        float q[8];
        block_codes(x, sb, q);
        if (!live || page < 0) continue;
        char * slab = slab0 + (size_t) h * S::BYTES, * at_v = slab + S::V + (slot >> 2) * 64 * NB + (i >> 2) * 4 + pm_kv4_vbyte(slot);
#pragma unroll
        for (int j = 0; j < 4; ++j) *(PM_G uint8_t *) (at_v + ((i & 3) * 4 + j) * 4 * NB) = (uint8_t) (uint32_t) fmaf(q[j + 4], 16.0f, q[j]);
        if ((i & 3) == 0) *(PM_G uint16_t *) (slab + S::VS + ((i >> 2) * PM_PAGE + slot) * 2) = sb;
    }
    if (n >= N) return;
    float w[8], ck[4], sk[4];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = a.wq ? a.wq[(j < 4 ? o0 : o1 - 4) + j] : 1.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) { ck[j] = turn ? (float) cs[i * 4 + j][0] : 1.0f; sk[j] = turn ? (float) cs[i * 4 + j][1] : 0.0f; }
    for (; n < N; n += parts) {
        const int h = (n - 2 * NG) * RPW + sub;
        const bool live = take(a.H, h);
        if (a.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
            const float mean = head_sum<LPH>(ss) * (1.0f / D) + a.eps, r = __builtin_amdgcn_rsqf(mean);      // (v_rsq_f32: 1 unit of 2^-23)
            // squares that leave 32 bits - values beyond 10^19, or below 10^-15 without an eps that says more - are summed in 64, like those of keys
            const bool odd = !(mean > 1e-30f && mean < 1e30f);
            if (__any(live && odd)) {
                double s2 = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) s2 = fma((double) x[j], (double) x[j], s2);
                const double r2 = 1.0 / sqrt(head_sum<LPH>(s2) / D + (double) a.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = odd ? (float) (x[j] * r2 * w[j]) : x[j] * (r * w[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= r * w[j];
            }
        }
        if (rot) {
            if (a.neox)
#pragma unroll
                for (int j = 0; j < 4; ++j) { const float u = x[j], v = x[j + 4]; x[j] = u * ck[j] - v * sk[j]; x[j + 4] = v * ck[j] + u * sk[j]; }
            else
#pragma unroll
                for (int j = 0; j < 4; ++j) { const float u = x[2 * j], v = x[2 * j + 1]; x[2 * j] = u * ck[j] - v * sk[j]; x[2 * j + 1] = v * ck[j] + u * sk[j]; }
        }
        if (live) { T * d = (T *) a.q + (size_t) t * a.ldq + h * D; st4(d + o0, x); st4(d + o1, x + 4); }
    }
}

// one (token, KV head) per LPH lanes
template <int NB> __global__ __launch_bounds__(256) void load_kernel(pm_kv4_cache c, const int32_t * pos, const int32_t * seq, int rows, _Float16 * k, _Float16 * v) {
    constexpr int D = NB * 32, LPH = NB <= 2 ? 8 : NB <= 4 ? 16 : 32;
    typedef pm_kv4_slab<NB> S;
    const int r = (blockIdx.x * 256 + threadIdx.x) / LPH, i = threadIdx.x % LPH;
    if (r >= rows || i * 8 >= D) return;
    const int t = r / c.G, h = r % c.G, page = pm_kv4_page(c, seq[t], pos[t]), slot = pos[t] & (PM_PAGE - 1), w = i >> 2, n = (i & 3) * 4;
    f16x8 x = {}, y = {};
    if (page >= 0) {
        const char * slab = c.pages + ((size_t) page * c.G + h) * S::BYTES;
        const uint32_t kc = *(const PM_G uint32_t *) (slab + S::K + slot * 16 * NB + (i & 3) * 4 * NB + w * 4);
        const _Float16 ks = *(const PM_G _Float16 *) (slab + S::KS + (slot * NB + w) * 2), vs = *(const PM_G _Float16 *) (slab + S::VS + (w * PM_PAGE + slot) * 2);
        const char * at_v = slab + S::V + (slot >> 2) * 64 * NB + w * 4 + pm_kv4_vbyte(slot);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = ks * (_Float16) ((int) (kc >> ((j & 1) * 16 + (j >> 1) * 4) & 15) - 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t b = *(const PM_G uint8_t *) (at_v + (n + j) * 4 * NB);
            y[j] = vs * (_Float16) ((int) (b & 15) - 8);
            y[j + 4] = vs * (_Float16) ((int) (b >> 4) - 8);
        }
    }
    *(PM_G f16x8 *) (k + (size_t) r * D + i * 8) = x;
    const u32x4 yy = __builtin_bit_cast(u32x4, y);
    *(PM_G u32x2 *) (v + (size_t) r * D + w * 32 + n) = u32x2{yy.x, yy.y};
    *(PM_G u32x2 *) (v + (size_t) r * D + w * 32 + n + 16) = u32x2{yy.z, yy.w};
}

} // namespace

#define PM_KV4_DIMS(CALL) switch (c.d) { case 64: CALL(2); break; case 96: CALL(3); break; case 128: CALL(4); break; case 192: CALL(6); break; case 256: CALL(8); break; default: return PM355_E_UNSUPPORTED; }

int pm_launch_kv4_append(const pm_kv4_cache & c, const pm_kv4_append & a, hipStream_t st) {
    // waves per token: one where tokens alone give every SIMD eight, down to one per group of head rows
    const int rpw = c.d <= 64 ? 8 : c.d <= 128 ? 4 : 2, groups = 2 * ((c.G + rpw - 1) / rpw) + (a.H + rpw - 1) / rpw, fill = 8192 / a.T;
    const int parts = fill < 1 ? 1 : fill < groups ? fill : groups;
    const int64_t blocks = ((int64_t) a.T * parts + 3) / 4;
    if (blocks >= 1 << 24) return PM355_E_SHAPE;           // (a launch has fewer than 2^32 threads)
#define PM_CALL(NB) \
    if (a.type == PM_BF16) hipLaunchKernelGGL((append_kernel<uint16_t, NB>), dim3((unsigned) blocks), dim3(256), 0, st, c, a, parts); \
    else hipLaunchKernelGGL((append_kernel<float, NB>), dim3((unsigned) blocks), dim3(256), 0, st, c, a, parts)
    PM_KV4_DIMS(PM_CALL)
#undef PM_CALL
    return 0;
}
int pm_launch_kv4_load(const pm_kv4_cache & c, const int32_t * pos, const int32_t * seq, int T, void * k, void * v, hipStream_t st) {
    const int lph = c.d <= 64 ? 8 : c.d <= 128 ? 16 : 32, rows = T * c.G;
#define PM_CALL(NB) hipLaunchKernelGGL(load_kernel<NB>, dim3((rows + 256 / lph - 1) / (256 / lph)), dim3(256), 0, st, c, pos, seq, rows, (_Float16 *) k, (_Float16 *) v)
    PM_KV4_DIMS(PM_CALL)
#undef PM_CALL
    return 0;
}
