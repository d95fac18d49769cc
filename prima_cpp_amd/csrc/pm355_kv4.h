// pm355_kv4.h — pages of a 4-bit KV cache (layout: include/prima_mi355.h): launch interface of kv4.hip, attn_kv4.hip and pages.hip, and the layout for their kernels.
#pragma once
#include "pm355_dense.h"

constexpr int PM_KV4_MAX_D = 256;
static inline bool pm_kv4_dim(int d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// slab of one KV head in a page, d = 32 nb: byte offsets of its four parts
template <int NB> struct pm_kv4_slab {
    static constexpr int CODES = PM_PAGE * 16 * NB, SCALES = PM_PAGE * 2 * NB, K = 0, KS = CODES, V = CODES + SCALES, VS = V + CODES, BYTES = VS + SCALES;
};
static inline size_t pm_kv4_slab_bytes(int d) { return (size_t) PM_PAGE * 36 * (d / 32); }

struct pm_kv4_cache { int G, d, n_pages; char * pages; const int32_t * table; int table_ld, n_seq; };
struct pm_kv4_append {
    int type, H, T; const void * proj; int64_t ldp; void * q; int64_t ldq;
    int norm; const float * wq, * wk; float eps; const double * turns; int n_rot, neox; float mscale;
    const int32_t * pos, * seq;
};
struct pm_kv4_attn {
    int type, H; const void * q; int64_t ldq; void * out; int64_t ldo;
    float scale; int window, first; const int32_t * tiles; int n_tiles, tile_tokens, max_keys, n_tokens;
    float * work; size_t work_floats;
};
int pm_launch_kv4_append(const pm_kv4_cache & c, const pm_kv4_append & a, hipStream_t st);
int pm_launch_kv4_load(const pm_kv4_cache & c, const int32_t * pos, const int32_t * seq, int T, void * k, void * v, hipStream_t st);
// what a call launches: columns of a workgroup (16, 32: few_kernel, 128: tiles_kernel), passes over the columns of a tile and how many of them start side by side, workgroups that share the keys of
// one, workgroups in all and whether a launch takes so many
struct pm_kv4_plan { int cols, passes, launched, splits; int64_t groups; bool fits; };
pm_kv4_plan pm_attn_kv4_plan(const pm_kv4_cache & c, const pm_kv4_attn & a);
int pm_launch_attn_kv4(const pm_kv4_cache & c, const pm_kv4_attn & a, hipStream_t st);
size_t pm_kv4_work_floats(int H, int G, int d);
int pm_launch_pages_copy(char * pages, size_t page_bytes, size_t layer_bytes, int n_layers, const int32_t * pairs, int n_pairs, hipStream_t st);

#ifdef __HIPCC__
// page of a position, -1 where none is held (whatever the caller's tables hold, nothing outside the pool is touched)
__device__ __forceinline__ int pm_kv4_page(const pm_kv4_cache & c, int seq, int pos) {
    if ((unsigned) seq >= (unsigned) c.n_seq || pos < 0 || pos / PM_PAGE >= c.table_ld) return -1;
    const int p = ld_g(c.table + (size_t) seq * c.table_ld + pos / PM_PAGE);
    return (unsigned) p < (unsigned) c.n_pages ? p : -1;
}
// place in a word of value codes: byte of a token in its quad
__device__ __forceinline__ int pm_kv4_vbyte(int token) { return (token & 1) * 2 + (token >> 1 & 1); }
#endif
