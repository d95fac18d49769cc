// kv4.hip — into a 4-bit KV cache and out of it: per-head norm of queries and keys, rotation, rounding to 4 bits, one pass over the projections.
//
// y = x / sqrt(mean(x^2) + eps) w;  (a, b) -> (a cos - b sin, b cos + a sin) mscale at 2 pi frac(pos turns_i);  scale = f16(M / -8), code = clamp(rint(y / scale), -8, 7) + 8.
// Bound by memory: a row of (H + 2 G) d values is read once, H d values and 1.125 G d bytes are written.
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include "../../include/prima_mi355.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void st4(float * p, const float * v) { *(PM_G f32x4 *) p = f32x4{v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void st4(uint16_t * p, const float * v) { *(PM_G u16x4 *) p = u16x4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])}; }

template <int LPH, typename F> __device__ __forceinline__ F head_sum(F v) {       // over the LPH lanes of a head row
#pragma unroll
    for (int m = 1; m < LPH; m *= 2) v += __shfl_xor(v, m);
    return v;
}
// scale (f16 bits) of a block whose 32 values lie in four neighbouring lanes, 8 each; NaN where the row holds a NaN or an infinity
template <int LPH> __device__ __forceinline__ uint16_t block_scale(const float * x, bool on) {
    float hi = -INFINITY, lo = INFINITY, bad = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { hi = fmaxf(hi, x[j]); lo = fminf(lo, x[j]); bad += on ? x[j] * 0.0f : 0.0f; }       // (0 * NaN, 0 * inf: NaN)
#pragma unroll
    for (int m = 1; m < 4; m *= 2) { hi = fmaxf(hi, __shfl_xor(hi, m)); lo = fminf(lo, __shfl_xor(lo, m)); }
    bad = head_sum<LPH>(bad);
    const float s = fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -8188.0f), 8188.0f);
    return bad == 0.0f ? f2h(s) : (uint16_t) 0x7e00;
}
__device__ __forceinline__ uint32_t code_of(float x, float s) {
    if (!(s != 0.0f) || !(s == s)) return 8;               // (an empty block, a row that is not finite)
    return (uint32_t) (int) (fminf(fmaxf(rintf(x / s), -8.0f), 7.0f) + 8.0f);
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
    for (int n = part; n < N; n += parts) {
        float x[8];
        widen(next, x);
        next = load(n + parts < N ? n + parts : n);
        const bool key = n < NG, val = !key && n < 2 * NG;
        const int h = (key ? n : val ? n - NG : n - 2 * NG) * RPW + sub;
        const bool live = on && h < (key || val ? G : a.H);
        if (!live)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.0f;
        if (!key && !val) {
            if (a.norm) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
                const float r = 1.0f / sqrtf(head_sum<LPH>(ss) / (float) D + a.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= r * (a.wq ? a.wq[(j < 4 ? o0 : o1 - 4) + j] : 1.0f);
            }
            if (turn)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float & p = a.neox ? x[j] : x[2 * j], & q = a.neox ? x[j + 4] : x[2 * j + 1];
                    const float k = (float) cs[i * 4 + j][0], s = (float) cs[i * 4 + j][1], u = p, v = q;
                    p = u * k - v * s; q = v * k + u * s;
                }
            if (live) { T * d = (T *) a.q + (size_t) t * a.ldq + h * D; st4(d + o0, x); st4(d + o1, x + 4); }
            continue;
        }
        char * slab = slab0 + (size_t) h * S::BYTES;
        if (val) {
            const uint16_t sb = block_scale<LPH>(x, live);
            const float s = h2f(sb);
            if (!live || page < 0) continue;
            char * at_v = slab + S::V + (slot >> 2) * 64 * NB + (i >> 2) * 4 + pm_kv4_vbyte(slot);
#pragma unroll
            for (int j = 0; j < 4; ++j) *(PM_G uint8_t *) (at_v + ((i & 3) * 4 + j) * 4 * NB) = (uint8_t) (code_of(x[j], s) | code_of(x[j + 4], s) << 4);
            if ((i & 3) == 0) *(PM_G uint16_t *) (slab + S::VS + ((i >> 2) * PM_PAGE + slot) * 2) = sb;
            continue;
        }
        // keys: 64 bits up to the one rounding to 32, so that a code never depends on the order of a sum
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
        if (live)
#pragma unroll
            for (int j = 0; j < 4; ++j) { kb[o0 + j] = (float) y[j]; kb[o1 + j] = (float) y[j + 4]; }
        lds_done();
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = live ? kb[i * 8 + j] : 0.0f;
        lds_done();
        const uint16_t sb = block_scale<LPH>(x, live);
        if (!live || page < 0) continue;
        const float s = h2f(sb);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= code_of(x[j], s) << ((j & 1) * 16 + (j >> 1) * 4);
        *(PM_G uint32_t *) (slab + S::K + slot * 16 * NB + (i & 3) * 4 * NB + (i >> 2) * 4) = w;
        if ((i & 3) == 0) *(PM_G uint16_t *) (slab + S::KS + (slot * NB + (i >> 2)) * 2) = sb;
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
    // waves per token: one where tokens alone give every SIMD two, down to one per group of head rows
    const int rpw = c.d <= 64 ? 8 : c.d <= 128 ? 4 : 2, groups = 2 * ((c.G + rpw - 1) / rpw) + (a.H + rpw - 1) / rpw, fill = 2048 / a.T;
    const int parts = fill < 1 ? 1 : fill < groups ? fill : groups;
    const int64_t blocks = ((int64_t) a.T * parts + 3) / 4;
    if (blocks > 0x3fffffff) return PM355_E_SHAPE;
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
