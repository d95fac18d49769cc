// kv4_api.hip — extern "C" surface of the 4-bit cache and of the page copies (part A"' of include/prima_mi355.h).
#include "../../include/prima_mi355.h"
#include "pm355_kv4.h"
#include "pm355_kernels.h"
#include <math.h>
#include <algorithm>
#include <new>
#include <vector>

static int fail(int code, const char * what) { return pm_api_fail(code, what, hipSuccess); }
static int done(int rc, const char * what) {
    if (rc) return fail(rc, what);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : pm_api_fail(PM355_E_HIP, what, e);
}
static bool aligned(const void * p, size_t n) { return (uintptr_t) p % n == 0; }
static bool known(int type) { return type == PM_BF16 || type == PM_F32; }
// null, or what is wrong with a cache
static const char * wrong(const pm355_kv4_cache * c) {
    if (!c || !c->pages || !c->d_table || c->n_pages < 1 || c->n_seq < 1 || c->table_ld < 1 || c->table_ld > 0x7fffffff / PM_PAGE) return "cache";
    if (c->n_head_kv < 1 || c->n_head_kv > 65535 || !pm_kv4_dim(c->head_dim)) return "n_head_kv, head_dim";
    return aligned(c->pages, 16) ? nullptr : "pages are not 16-byte aligned";
}
static pm_kv4_cache cache_of(const pm355_kv4_cache * c) { return {c->n_head_kv, c->head_dim, c->n_pages, (char *) c->pages, c->d_table, c->table_ld, c->n_seq}; }
// the launch's arguments of a call of attn_kv4, or the code of what is wrong with it
static int attn_of(const pm355_kv4_cache * c, const pm355_attn_kv4_args * p, pm_kv4_attn & a) {
    if (const char * w = wrong(c)) return fail(PM355_E_SHAPE, w);
    const int64_t d = c->head_dim;
    if (!p || !known(p->type)) return fail(PM355_E_UNSUPPORTED, "attn_kv4: type");
    a = {p->type, p->n_head, p->q, p->ldq, p->out, p->ldo, p->scale, p->window, p->n_first, p->d_tiles, p->n_tiles, p->tile_tokens, p->max_keys, p->n_tokens, p->work, p->work ? p->work_floats : 0};
    if (p->n_tiles == 0) return 0;
    if (p->n_tiles < 0 || p->n_tokens < 1 || p->n_head < 1 || p->n_head % c->n_head_kv || !p->q || !p->out || !p->d_tiles || p->ldq < p->n_head * d || p->ldo < p->n_head * d || p->n_head * d > 0x0fffffff ||
        p->window < 0 || p->n_first < 0 || p->max_keys < 0)
        return fail(PM355_E_SHAPE, "attn_kv4: shape");
    if (p->tile_tokens < 1 || (p->tile_tokens > 1 && (int64_t) p->n_head / c->n_head_kv * p->tile_tokens > 128)) return fail(PM355_E_SHAPE, "attn_kv4: tile_tokens");
    if (!isfinite(p->scale)) return fail(PM355_E_RANGE, "attn_kv4: scale");
    if ((int64_t) p->n_tiles * p->tile_tokens > 0x7fffffff) return fail(PM355_E_SHAPE, "attn_kv4: n_tiles");
    if (p->ldq % 8 || p->ldo % 8 || !aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->d_tiles, 16) || !aligned(p->work, 16)) return fail(PM355_E_ALIGN, "attn_kv4: rows");
    return 0;
}

extern "C" {

size_t pm355_kv4_page_bytes(int n_head_kv, int head_dim) { return n_head_kv > 0 && pm_kv4_dim(head_dim) ? n_head_kv * pm_kv4_slab_bytes(head_dim) : 0; }

int pm355_kv4_append(const pm355_kv4_cache * c, const pm355_kv4_append_args * p, pm355_stream_t st) {
    if (const char * w = wrong(c)) return fail(PM355_E_SHAPE, w);
    const int d = c->head_dim;
    if (!p || !known(p->type)) return fail(PM355_E_UNSUPPORTED, "kv4_append: type");
    if (p->n_tokens == 0) return 0;
    if (p->n_tokens < 0 || p->n_head < 1 || p->n_head % c->n_head_kv || !p->proj || !p->q || !p->d_pos || !p->d_seq || p->ld_proj < ((int64_t) p->n_head + 2 * c->n_head_kv) * d ||
        p->ldq < (int64_t) p->n_head * d || (int64_t) p->n_head * d > 0x0fffffff)
        return fail(PM355_E_SHAPE, "kv4_append: shape");
    if (p->d_turns && (p->n_rot < 8 || p->n_rot % 8 || p->n_rot > d)) return fail(PM355_E_SHAPE, "kv4_append: n_rot");
    if (!isfinite(p->mscale) || !isfinite(p->eps)) return fail(PM355_E_RANGE, "kv4_append: mscale, eps");
    if (p->ld_proj % 4 || p->ldq % 4 || !aligned(p->proj, 16) || !aligned(p->q, 16)) return fail(PM355_E_ALIGN, "kv4_append: rows");
    (void) hipGetLastError();
    return done(pm_launch_kv4_append(cache_of(c), {p->type, p->n_head, p->n_tokens, p->proj, p->ld_proj, p->q, p->ldq, p->norm, p->norm_q, p->norm_k, p->eps, p->d_turns, p->n_rot, p->rope_neox, p->mscale,
                                                   p->d_pos, p->d_seq}, (hipStream_t) st), "kv4_append");
}

int pm355_kv4_load(const pm355_kv4_cache * c, const int32_t * d_pos, const int32_t * d_seq, int n_tokens, void * k, void * v, pm355_stream_t st) {
    if (const char * w = wrong(c)) return fail(PM355_E_SHAPE, w);
    if (n_tokens == 0) return 0;
    if (n_tokens < 0 || !d_pos || !d_seq || !k || !v || (int64_t) n_tokens * c->n_head_kv * 32 > 0x7fffffff) return fail(PM355_E_SHAPE, "kv4_load: shape");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(PM355_E_ALIGN, "kv4_load: rows");
    (void) hipGetLastError();
    return done(pm_launch_kv4_load(cache_of(c), d_pos, d_seq, n_tokens, k, v, (hipStream_t) st), "kv4_load");
}

int pm355_rope_turns(const pm355_rope_params * rp, const float * freq_factors, double * turns, float * mscale) {
    if (!rp || !turns || !mscale || rp->n_dims < 2 || rp->n_dims % 2 || !(rp->freq_base > 0.0f)) return fail(PM355_E_SHAPE, "rope_turns: shape");
    const double n = rp->n_dims, base = rp->freq_base;
    auto corr = [&](double rotations) { return n * log(rp->n_ctx_orig / (rotations * 2 * M_PI)) / (2 * log(base)); };
    const double lo = rp->ext_factor != 0.0f ? fmax(0.0, floor(corr(rp->beta_fast))) : 0.0, hi = rp->ext_factor != 0.0f ? fmin(n - 1, ceil(corr(rp->beta_slow))) : 0.0;
    for (int i = 0; i < rp->n_dims / 2; ++i) {
        const double t = pow(base, -2.0 * i / n) / (2 * M_PI) / (freq_factors ? freq_factors[i] : 1.0);
        const double mix = rp->ext_factor != 0.0f ? rp->ext_factor * (1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(0.001, hi - lo)))) : 0.0;
        turns[i] = t * rp->freq_scale * (1.0 - mix) + t * mix;
    }
    *mscale = rp->ext_factor != 0.0f ? (float) (rp->attn_factor * (1.0 + 0.1 * log(1.0 / rp->freq_scale))) : rp->attn_factor;
    return 0;
}

size_t pm355_attn_kv4_work_floats(int n_head, int n_head_kv, int head_dim) {
    return n_head_kv > 0 && n_head > 0 && n_head % n_head_kv == 0 && pm_kv4_dim(head_dim) ? pm_kv4_work_floats(n_head, n_head_kv, head_dim) : 0;
}
int pm355_attn_kv4(const pm355_kv4_cache * c, const pm355_attn_kv4_args * p, pm355_stream_t st) {
    pm_kv4_attn a;
    if (const int rc = attn_of(c, p, a)) return rc;
    if (a.n_tiles == 0) return 0;
    (void) hipGetLastError();
    return done(pm_launch_attn_kv4(cache_of(c), a, (hipStream_t) st), "attn_kv4");
}
int pm355_attn_kv4_plan(const pm355_kv4_cache * c, const pm355_attn_kv4_args * p, int32_t * out4) {
    pm_kv4_attn a;
    if (!out4) return fail(PM355_E_SHAPE, "attn_kv4_plan: out4");
    if (const int rc = attn_of(c, p, a)) return rc;
    const pm_kv4_plan pl = a.n_tiles ? pm_attn_kv4_plan(cache_of(c), a) : pm_kv4_plan{0, 0, 0, 0, 0, true};
    if (!pl.fits) return fail(PM355_E_SHAPE, "attn_kv4: n_tiles");
    out4[0] = pl.cols; out4[1] = pl.launched; out4[2] = pl.splits; out4[3] = (int32_t) pl.groups;
    return 0;
}

int pm355_pages_copy(void * pages, size_t page_bytes, size_t layer_bytes, int n_layers, int n_pages, const int32_t * pairs, int n_pairs, pm355_stream_t st) {
    if (n_pairs == 0) return 0;
    if (!pages || !pairs || n_pairs < 0 || n_pairs > n_pages || n_pages > 0x3fffffff || n_layers < 1 || n_pages < 1 || page_bytes < 16 || page_bytes > (size_t) 1 << 32 || (n_layers > 1 && layer_bytes / page_bytes < (size_t) n_pages))
        return fail(PM355_E_SHAPE, "pages_copy: shape");
    if (page_bytes % 16 || layer_bytes % 16 || !aligned(pages, 16)) return fail(PM355_E_ALIGN, "pages_copy: pages");
    try {
        std::vector<unsigned char> is((size_t) n_pages);                    // 1: read, 2: written
        for (int i = 0; i < 2 * n_pairs; ++i) if ((unsigned) pairs[i] >= (unsigned) n_pages) return fail(PM355_E_RANGE, "pages_copy: page");
        for (int i = 0; i < n_pairs; ++i) is[pairs[2 * i]] = 1;
        for (int i = 0; i < n_pairs; ++i) { if (is[pairs[2 * i + 1]]) return fail(PM355_E_RANGE, "pages_copy: a page is copied to twice, or copied to and from"); is[pairs[2 * i + 1]] = 2; }
    } catch (...) { return fail(PM355_E_NOMEM, "pages_copy"); }
    (void) hipGetLastError();
    return done(pm_launch_pages_copy((char *) pages, page_bytes, layer_bytes, n_layers, pairs, n_pairs, (hipStream_t) st), "pages_copy");
}

} // extern "C"
