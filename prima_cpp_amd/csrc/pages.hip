// pages.hip — pages of a pool copied in every layer. Bound by memory: every byte is read and written once, 16 per lane. 501 pages of 72 KB in 8 layers 123 us (591 MB, 4.8 TB/s; a copy of 2 GB
// 4.9), one page in 16 layers 2.9 us.
#include "pm355_kv4.h"
#include "../../include/prima_mi355.h"

namespace {

// (from, to) pairs as a kernel argument: nothing to allocate, nothing that a captured graph could share or outlive
constexpr int PAIRS = 448;
struct pairs_arg { int32_t at[PAIRS][2]; };
static_assert(sizeof(pairs_arg) <= 3584, "kernel arguments are at most 4 KB");

constexpr int PIECE = 4;                                   // 16-byte loads in flight per lane
__global__ __launch_bounds__(256) void pages_copy_kernel(char * pages, size_t page_bytes, size_t layer_bytes, pairs_arg p) {
    char * layer = pages + (size_t) blockIdx.z * layer_bytes;
    const char * src = layer + (size_t) p.at[blockIdx.y][0] * page_bytes;
    char * dst = layer + (size_t) p.at[blockIdx.y][1] * page_bytes;
    const size_t o = ((size_t) blockIdx.x * 256 * PIECE + threadIdx.x) * 16;
    u32x4 v[PIECE];
#pragma unroll
    for (int j = 0; j < PIECE; ++j) if (o + j * 4096 < page_bytes) v[j] = *(const PM_G u32x4 *) (src + o + j * 4096);
#pragma unroll
    for (int j = 0; j < PIECE; ++j) if (o + j * 4096 < page_bytes) *(PM_G u32x4 *) (dst + o + j * 4096) = v[j];
}

} // namespace

int pm_launch_pages_copy(char * pages, size_t page_bytes, size_t layer_bytes, int n_layers, const int32_t * pairs, int n_pairs, hipStream_t st) {
    for (int at = 0; at < n_pairs; at += PAIRS) {
        const int n = n_pairs - at < PAIRS ? n_pairs - at : PAIRS;
        pairs_arg p{};
        for (int i = 0; i < n; ++i) { p.at[i][0] = pairs[2 * (at + i)]; p.at[i][1] = pairs[2 * (at + i) + 1]; }
        for (int l = 0; l < n_layers; l += 32768) {
            const int nl = n_layers - l < 32768 ? n_layers - l : 32768;
            hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned) ((page_bytes + 256 * PIECE * 16 - 1) / (256 * PIECE * 16)), n, nl), dim3(256), 0, st, pages + (size_t) l * layer_bytes, page_bytes,
                               layer_bytes, p);
        }
    }
    return 0;
}
