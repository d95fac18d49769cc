// attn_kv4.hip — attention over pages held in 4 bits: causal, with a sliding window and first tokens that stay visible.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q k_j - max), over the j that the query sees; one pass over the keys with the running maximum and sum.
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include "../../include/prima_mi355.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -1e30f;                             // running maximum before the first visible key

// one (token, head) per workgroup on the vector pipe: a lane per key for the scores, a lane per dimension for the values
template <typename T, int NB> __global__ __launch_bounds__(256) void attn_kernel(pm_kv4_cache c, pm_kv4_attn a) {
    constexpr int D = NB * 32;
    typedef pm_kv4_slab<NB> S;
    __shared__ float q[D], acc[4][D], p[4][PM_PAGE], ml[4][2];
    const int32_t * tile = a.tiles + blockIdx.x / a.tile_tokens * 4;
    const int i = blockIdx.x % a.tile_tokens, h = blockIdx.y, g = h / (a.H / c.G), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (i >= tile[1] || (unsigned) (tile[0] + i) >= (unsigned) a.n_tokens) return;
    const int t = tile[0] + i, pos = tile[2] < 0 ? -1 : tile[2] + i, seq = tile[3];
    for (int d = threadIdx.x; d < D; d += 256) { q[d] = to_f<T>(((const T *) a.q)[(size_t) t * a.ldq + h * D + d]) * a.scale; for (int w = 0; w < 4; ++w) acc[w][d] = 0.0f; }
    __syncthreads();
    float m = NONE, l = 0.0f;
    for (int pg = wave; pg <= (pos < 0 ? -1 : pos / PM_PAGE); pg += 4) {
        const int page = pm_kv4_page(c, seq, pg * PM_PAGE), key = pg * PM_PAGE + lane;
        if (page < 0) continue;
        const char * slab = c.pages + ((size_t) page * c.G + g) * S::BYTES;
        const bool ok = key <= pos && (a.window <= 0 || pos - key < a.window || key < a.first);
        float s = 0.0f;
        for (int b = 0; b < NB; ++b) {
            const float ks = h2f(*(const PM_G uint16_t *) (slab + S::KS + (lane * NB + b) * 2));
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = *(const PM_G uint32_t *) (slab + S::K + lane * 16 * NB + e * 4 * NB + b * 4);
                for (int j = 0; j < 8; ++j) s = fmaf(q[b * 32 + e * 8 + j], h2f(f2h(ks * (float) ((int) (w >> ((j & 1) * 16 + (j >> 1) * 4) & 15) - 8))), s);
            }
        }
        const float mn = fmaxf(m, wave_max(ok ? s : NONE)), e = ok ? expf(s - mn) : 0.0f, corr = expf(m - mn);
        l = l * corr + wave_sum(e); m = mn;
        p[wave][lane] = e;
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int d = lane; d < D; d += 64) {
            const int b = d / 32, n = d % 16, hi = d / 16 % 2;
            float o = acc[wave][d] * corr;
            for (int j = 0; j < PM_PAGE; ++j) {
                const uint32_t w = *(const PM_G uint8_t *) (slab + S::V + (j >> 2) * 64 * NB + n * 4 * NB + b * 4 + pm_kv4_vbyte(j));
                const float v = h2f(f2h(h2f(*(const PM_G uint16_t *) (slab + S::VS + (b * PM_PAGE + j) * 2)) * (float) ((int) (w >> 4 * hi & 15) - 8)));
                if (p[wave][j] != 0.0f) o = fmaf(p[wave][j], v, o);
            }
            acc[wave][d] = o;
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) { ml[wave][0] = m; ml[wave][1] = l; }
    __syncthreads();
    float M = NONE, L = 0.0f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w][0]);
    for (int w = 0; w < 4; ++w) L += ml[w][1] * expf(ml[w][0] - M);
    for (int d = threadIdx.x; d < D; d += 256) {
        float o = 0.0f;
        for (int w = 0; w < 4; ++w) o += acc[w][d] * expf(ml[w][0] - M);
        ((T *) a.out)[(size_t) t * a.ldo + h * D + d] = from_f<T>(L == 0.0f ? 0.0f : o / L);
    }
}

} // namespace

size_t pm_kv4_work_floats(int H, int G, int d) { return 0; }
int pm_launch_attn_kv4(const pm_kv4_cache & c, const pm_kv4_attn & a, hipStream_t st) {
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(a.n_tiles * a.tile_tokens, a.H), dim3(256), 0, st, c, a); return 0; };
#define PM_CALL(NB) return a.type == PM_BF16 ? go(attn_kernel<uint16_t, NB>) : go(attn_kernel<float, NB>)
    switch (c.d) { case 64: PM_CALL(2); case 96: PM_CALL(3); case 128: PM_CALL(4); case 192: PM_CALL(6); case 256: PM_CALL(8); }
    return PM355_E_UNSUPPORTED;
}
