// okf_attn.hip -- the C ABI of attention and the KV cache (include/okf_quant.h)
// over okf_attn.h, okf_attn_dec.h and okf_kv.h.
#include "okf_impl.h"
#include "okf_args.h"
#include "okf_attn_run.h"
#include "okf_attn_dec.h"
#include "okf_kv.h"

namespace {

using namespace okf;
using namespace okf_impl;

// Runs f with the 64s of dimensions that hold dim, as a constant.
template <class Fn>
void with_dims(uint32_t dim, Fn f) {
    switch ((dim + 63) / 64) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    default: f(std::integral_constant<int, 4>{}); break;
    }
}

int check_cache(const okf_kv_cache *c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return OKF_E_ARG;
    if (!c->pages || c->pages > 0x7FFFFFFFu || !c->heads || c->heads > 65535 || !good_dim(c->dim)) return OKF_E_SHAPE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned4(c->k_scale) || !aligned4(c->v_scale)) return OKF_E_SHAPE;
    return OKF_OK;
}

int check_seqs(const okf_kv_seqs *s) {
    if (!s || !s->pages || !s->len) return OKF_E_ARG;
    if (!s->count || !s->stride || !aligned4(s->pages) || !aligned4(s->len)) return OKF_E_SHAPE;
    return OKF_OK;
}

KvCache cache_of(const okf_kv_cache *c) { return {c->k, c->v, c->k_scale, c->v_scale, c->pages, c->heads, c->dim}; }
KvSeqs seqs_of(const okf_kv_seqs *s) { return {s->pages, s->len, s->count, s->stride}; }

// Whether n rows of la values, sa apart, share memory with n rows of lb values, sb apart.
bool rows_meet(const float *a, uint64_t sa, uint64_t la, const float *b, uint64_t sb, uint64_t lb, uint64_t n) {
    const uint64_t pa = (uint64_t)(uintptr_t)a / sizeof(float), pb = (uint64_t)(uintptr_t)b / sizeof(float);
    if (pa + (n - 1) * sa + la <= pb || pb + (n - 1) * sb + lb <= pa) return false;
    for (uint64_t i = 0, j = 0; i < n && j < n;) {
        if (pa + i * sa + la <= pb + j * sb) i++;
        else if (pb + j * sb + lb <= pa + i * sa) j++;
        else return true;
    }
    return false;
}

// Arguments that okf_kv_append and okf_kv_read share, and their grid: n rows of
// `count` sequences touch at most n / 64 + 2 count page blocks.
int check_rows(const okf_kv_cache *c, const okf_kv_seqs *s, const void *k, const void *v, int32_t type,
               const int32_t *start, uint32_t n, uint64_t &ks, uint64_t &vs, dim3 &grid) {
    int st = check_cache(c);
    if (!st) st = check_seqs(s);
    if (st) return st;
    if (!start) return OKF_E_ARG;
    if (!attn_type(type)) return OKF_E_TYPE;
    const uint32_t size = type == F32 ? 4 : 2;
    if (!n || n > 0x7FFFFFFFu || !aligned16(k) || !aligned16(v) || !aligned4(start)) return OKF_E_SHAPE;
    const uint64_t row = (uint64_t)c->heads * c->dim;
    if (!row_stride(ks, row, size) || !row_stride(vs, row, size)) return OKF_E_SHAPE;
    const uint64_t items = n / KV_B + 3ull * s->count;
    if (items > 0xFFFFFFull) return OKF_E_SHAPE;  // (a grid has less than 2^32 threads)
    grid = dim3((uint32_t)items, c->heads, 2);
    return OKF_OK;
}

// The splits of okf_attn_decode: how many page ranges each sequence and kv head is cut
// into.  So many that the workgroups fill the CUs (as many at a time on each as the kernel's
// registers leave room for: two for up to 128 dimensions, one past that), but with a page
// for each of a workgroup's wavefronts, and two where that would be more workgroups than CUs
// (one sequence of 40000 tokens x 2 kv heads: 15.5 us, with one page 17.6; 1999 tokens x 8, 64
// workgroups: 12.3, with one page 10.8).  Batches of ragged sequences get up to twice that, so
// that the short ones' workgroups make room for the long ones', where four pages are left for
// each wavefront (32 of up to 8192 tokens 69 us, without 75; 20 of up to 3000 x 8 kv heads of
// 96 with weights 29, without 26).  The partial results go to the context's buffer; where it
// may not grow, as many splits as it holds.
constexpr uint64_t DEC_KEPT = 256ull << 20;  // bytes of scores at most
uint64_t up(uint64_t x, uint64_t y) { return (x + y - 1) / y; }

// The query rows of a kv head in blocks of 16 or 32, all sequences' and kv heads' blocks, and the
// workgroups that fill the CUs.
struct DecRows {
    uint64_t rows, rpb, rb, base, want;
    DecRows(const okf_ctx *c, uint64_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t tokens)
        : rows((uint64_t)tokens * (heads / kv_heads)), rpb(rows > 16 ? 32 : 16), rb(up(rows, rpb)), base(seqs * kv_heads * rb),
          want((uint64_t)c->cus * (dim <= 128 ? 2 : 1)) {}
    // bytes of scratch for n workgroups: maxima and sums, and the partial outputs of several splits
    uint64_t bytes(uint64_t n, uint32_t dim, bool several) const { return n * rpb * (2 + (several ? dim : 0)) * sizeof(float); }
};

// Bytes of the scores that are kept for the weights of up to `rows` query rows of a kv head, 0 where
// that is not less to write and read than the keys are to read again (8 sequences of up to 16000
// tokens, 2 rows of 64: 31.6 us without); more than DEC_KEPT are not kept.
uint64_t dec_kept(uint64_t heads, uint64_t rows, uint32_t dim, uint64_t stride) {
    if (rows > 16 || 8 * rows > dim) return 0;
    const uint64_t each = stride * KV_B * sizeof(float);
    return heads * rows > DEC_KEPT / each ? DEC_KEPT + 1 : heads * rows * each;
}

int plan_decode(okf_ctx *c, DecArgs &a) {
    const DecRows r(c, a.s.count, a.heads, a.c.heads, a.c.dim, a.tokens);
    a.rb = (uint32_t)r.rb;
    const uint64_t span = a.window ? std::min<uint64_t>(((uint64_t)a.window + a.tokens) / KV_B + 2, a.s.stride) : a.s.stride;
    const uint64_t each = r.base * up(span, DEC_W) <= c->cus ? 1 : 2;
    uint64_t splits = std::min(up(r.want, r.base), up(span, each * DEC_W));
    if (a.s.count > 1) splits = std::max(splits, std::min(up(2 * r.want, r.base), up(span, 4 * DEC_W)));
    splits = std::min<uint64_t>(splits, DEC_SPLITS);
    auto bytes = [&](uint64_t n) { return r.bytes(r.base * n, a.c.dim, n > 1); };
    const uint64_t kept = a.w_out ? dec_kept(r.base, r.rows, a.c.dim, a.s.stride) : 0, to = up(bytes(splits), 16) * 16;
    if (kept && kept <= DEC_KEPT && (to + kept <= c->part_bytes || grow_part(c, to + kept, true) == OKF_OK))
        a.sc = c->part + to / sizeof(float);
    else if (splits > 1 || a.w_out) {
        // (o over q: written by a launch behind the one that reads q again for the weights)
        const uint64_t least = a.w_out && a.q == a.o ? 2 : 1;
        splits = std::max(splits, least);
        if (bytes(splits) > c->part_bytes && grow_part(c, bytes(splits), true) != OKF_OK) {
            while (splits > least && bytes(splits) > c->part_bytes) splits--;
            if (a.w_out && bytes(splits) > c->part_bytes) return OKF_E_SHAPE;
        }
    }
    a.splits = (uint32_t)splits;
    if (splits > 1 || a.w_out) {
        a.ml = c->part;
        a.part = c->part + r.base * splits * r.rpb * 2;
    }
    if (r.base * splits + 8 * r.rb > 0xFFFFFFull || (splits > 1 && r.base / r.rb * r.rows > 0xFFFFFFull)) return OKF_E_SHAPE;
    return OKF_OK;
}

template <int KS, int NR>
void launch_decode_n(okf_ctx *c, const DecArgs &a) {
    static std::atomic<uint64_t> attr{0};
    set_lds_attr(c, (const void *)attn_dec_kernel<KS, NR>, attr);
    const uint32_t sh = a.s.count * a.c.heads;
    const size_t lds = (size_t)DEC_W * 16 * (a.c.dim + 4 + 2) * sizeof(float);
    hipLaunchKernelGGL((attn_dec_kernel<KS, NR>), dim3((sh * a.splits + 7) / 8 * 8 * a.rb), dim3(DEC_NT), lds, c->stream, a);
    const uint32_t joins = a.splits > 1 ? sh * a.tokens * (a.heads / a.c.heads) : 0;
    if (a.sc) {
        const uint32_t parts = std::max(1u, std::min(8 * c->cus / sh, (a.s.stride * KV_B + DEC_NT - 1) / DEC_NT));
        hipLaunchKernelGGL(attn_dec_sum_kernel, dim3(joins + sh * parts), dim3(DEC_NT), 0, c->stream, a, parts, joins);
    } else if (a.w_out) {
        const uint32_t parts = std::max(1u, std::min(4 * c->cus / sh, (a.s.stride + DEC_W - 1) / DEC_W));
        const uint32_t beside = a.q == a.o ? 0 : joins;
        hipLaunchKernelGGL((attn_dec_weights_kernel<KS, NR>), dim3(beside + sh * parts), dim3(DEC_NT), 0, c->stream, a, parts, beside);
        if (beside) return;
    }
    if (joins && !a.sc) hipLaunchKernelGGL(attn_dec_join_kernel, dim3(joins), dim3(DEC_NT), 0, c->stream, a, 16u * NR);
}

template <int KS>
void launch_decode(okf_ctx *c, const DecArgs &a, bool two) {
    two ? launch_decode_n<KS, 2>(c, a) : launch_decode_n<KS, 1>(c, a);
}

}  // namespace

extern "C" {

int okf_attn_prompt(okf_ctx *c, const okf_attn *p) {
    if (!p || !p->q || !p->k || !p->v || !p->o || !p->q_start || !p->k_start) return OKF_E_ARG;
    if (!attn_type(p->type)) return OKF_E_TYPE;
    if (!p->heads || !p->kv_heads || p->heads % p->kv_heads || p->heads > 65535 || !good_dim(p->dim)) return OKF_E_SHAPE;
    // (rows are counted in 32 bits with a sign, up to a workgroup's past the last)
    if (!p->seqs || !p->n_q || !p->n_k || p->n_q > 0x7FFFFF00u || p->n_k > 0x7FFFFF00u) return OKF_E_SHAPE;
    const uint32_t size = p->type == F32 ? 4 : 2;
    AttnArgs a{p->q, p->k, p->v, p->o, p->heads, p->kv_heads, p->dim, p->seqs, p->n_q, p->n_k, p->q_start, p->k_start,
               p->q_stride, p->k_stride, p->v_stride, p->o_stride, p->q_head, p->k_head, p->v_head, p->o_head,
               p->scale, p->window, 0};
    // (rows may lie inside a head's plane, heads inside a row: either stride may be the larger)
    const uint64_t least = p->dim;
    if (!a.qs) a.qs = (uint64_t)p->heads * p->dim;
    if (!a.os) a.os = (uint64_t)p->heads * p->dim;
    if (!a.ks) a.ks = (uint64_t)p->kv_heads * p->dim;
    if (!a.vs) a.vs = (uint64_t)p->kv_heads * p->dim;
    for (uint64_t *s : {&a.qs, &a.ks, &a.vs, &a.os, &a.qh, &a.kh, &a.vh, &a.oh})
        if (!row_stride(*s, least, size)) return OKF_E_SHAPE;
    if (a.ks > 1u << 23 || a.vs > 1u << 23) return OKF_E_SHAPE;  // (a tile's rows are addressed by 32-bit offsets)
    if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->o) || !aligned4(p->q_start) ||
        !aligned4(p->k_start))
        return OKF_E_SHAPE;
    int st = begin(c);
    if (st) return st;
    if (p->type == F32) st = launch_prompt<float>(c, a);
    else if (p->type == F16) st = launch_prompt<_Float16>(c, a);
    else st = launch_prompt<__bf16>(c, a);
    return st ? st : finish(c);
}

int okf_attn_decode(okf_ctx *c, const okf_kv_cache *cache, const okf_kv_seqs *seqs, const float *q, float *o,
                    uint32_t tokens, uint32_t heads, float scale, uint32_t window, const float *w_in, float *w_out,
                    uint64_t w_stride) {
    int st = check_cache(cache);
    if (!st) st = check_seqs(seqs);
    if (st) return st;
    if (!q || !o || (w_in && !w_out)) return OKF_E_ARG;
    if (!tokens || tokens > 65535 || !heads || heads % cache->heads || heads > 65535) return OKF_E_SHAPE;
    if (!aligned16(q) || !aligned16(o) || !aligned4(w_in) || !aligned4(w_out)) return OKF_E_SHAPE;
    if (w_out && w_stride < (uint64_t)seqs->stride * KV_B) return OKF_E_SHAPE;
    const uint64_t sh = (uint64_t)seqs->count * cache->heads, rows = (uint64_t)tokens * (heads / cache->heads);
    if (sh * rows > 0x3FFFFFFFull) return OKF_E_SHAPE;
    const uint64_t values = sh * rows * cache->dim;
    if (q != o && rows_meet(q, values, values, o, values, values, 1)) return OKF_E_ARG;
    const uint64_t row = (uint64_t)seqs->stride * KV_B;
    if (w_in && w_in != w_out && rows_meet(w_in, w_stride, row, w_out, w_stride, row, sh)) return OKF_E_ARG;
    if ((st = begin(c))) return st;
    DecArgs a{cache_of(cache), seqs_of(seqs), q, o, tokens, heads, scale, window, w_in, w_out, w_stride, 1, 1,
              nullptr, nullptr, nullptr};
    if ((st = plan_decode(c, a))) return st;
    if (a.ml) note_capture(c, false, true, false);
    with_dims(cache->dim, [&](auto ks) { launch_decode<decltype(ks)::value>(c, a, rows > 16); });
    return finish(c);
}

int okf_attn_reserve(okf_ctx *c, uint32_t seqs, uint32_t stride, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                     uint32_t tokens, int32_t weights) {
    if (!c) return OKF_E_ARG;
    if (!seqs || !stride || !tokens || tokens > 65535 || !heads || heads > 65535 || !kv_heads || heads % kv_heads || !good_dim(dim))
        return OKF_E_SHAPE;
    const uint64_t sh = (uint64_t)seqs * kv_heads, group = heads / kv_heads;
    if (sh * tokens * group > 0x3FFFFFFFull) return OKF_E_SHAPE;
    if (c->device < 0) return OKF_E_NODEV;
    (void)hipSetDevice(c->device);
    // Of any smaller call, too: base blocks in up(2 want, base) splits are less than 2 want + base
    // workgroups, and in a split for every DEC_W pages no more than that many (two splits at least
    // for weights with o over q); the scores are most with as many tokens as they are still kept for.
    const DecRows r(c, seqs, heads, kv_heads, dim, tokens);
    const uint64_t n = std::max(std::min(2 * r.want + r.base, r.base * up(stride, DEC_W)), weights ? 2 * r.base : 0);
    uint64_t need = up(r.bytes(n, dim, true), 16) * 16;
    const uint64_t most = std::min<uint64_t>(tokens, std::min(16u, dim / 8) / group);
    if (weights && most) need += std::min(dec_kept(sh, most * group, dim, stride), DEC_KEPT);
    const bool reserved = c->reserved;
    c->reserved = false;
    const int st = grow_part(c, need);
    c->reserved = reserved;
    return st;
}

int okf_kv_append(okf_ctx *c, const okf_kv_cache *cache, const okf_kv_seqs *seqs, const void *k, const void *v,
                  int32_t type, const int32_t *start, uint32_t n, uint64_t k_stride, uint64_t v_stride) {
    if (!k || !v) return OKF_E_ARG;
    dim3 grid;
    int st = check_rows(cache, seqs, k, v, type, start, n, k_stride, v_stride, grid);
    if (st) return st;
    if ((st = begin(c))) return st;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_dims(cache->dim, [&](auto nd) {
            hipLaunchKernelGGL((kv_append_kernel<T, decltype(nd)::value>), grid, dim3(KV_NT), 0, c->stream, cache_of(cache),
                               seqs_of(seqs), (const T *)k, (const T *)v, start, n, k_stride, v_stride);
        });
    });
    return finish(c);
}

int okf_kv_read(okf_ctx *c, const okf_kv_cache *cache, const okf_kv_seqs *seqs, void *k, void *v, int32_t type,
                const int32_t *start, uint32_t n, uint64_t k_stride, uint64_t v_stride) {
    if (!k && !v) return OKF_E_ARG;
    dim3 grid;
    int st = check_rows(cache, seqs, k, v, type, start, n, k_stride, v_stride, grid);
    if (st) return st;
    if ((st = begin(c))) return st;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_dims(cache->dim, [&](auto nd) {
            hipLaunchKernelGGL((kv_read_kernel<T, decltype(nd)::value>), grid, dim3(KV_NT), 0, c->stream, cache_of(cache),
                               seqs_of(seqs), (T *)k, (T *)v, start, n, k_stride, v_stride);
        });
    });
    return finish(c);
}

int okf_kv_evict(okf_ctx *c, const okf_kv_cache *src, const okf_kv_seqs *from, const okf_kv_cache *dst,
                 const okf_kv_seqs *to, uint32_t keep, uint32_t sink, uint32_t recent, const float *w_in,
                 uint64_t w_in_stride, float *w_out, uint64_t w_out_stride, int32_t *kept) {
    int st = check_cache(src);
    if (!st) st = check_seqs(from);
    if (!st) st = check_cache(dst);
    if (!st) st = check_seqs(to);
    if (st) return st;
    if (!w_in || !kept) return OKF_E_ARG;
    if (src->heads != dst->heads || src->dim != dst->dim || from->count != to->count) return OKF_E_SHAPE;
    if (!keep || keep > 0x7FFFFFFFu || (uint64_t)sink + recent > keep || keep > (uint64_t)to->stride * KV_B)
        return OKF_E_SHAPE;
    if (w_in_stride < (uint64_t)from->stride * KV_B || (w_out && w_out_stride < keep)) return OKF_E_SHAPE;
    if (!aligned4(w_in) || !aligned4(w_out) || !aligned4(kept)) return OKF_E_SHAPE;
    const uint64_t rows = (uint64_t)from->count * src->heads;
    if (rows > 0x3FFFFFull || keep > 0x3FFFFFFFu) return OKF_E_SHAPE;  // (grids of less than 2^32 threads)
    // (the second grid: sequences over y, in groups that fit it, and z)
    const uint32_t group = std::min(from->count, 65535 / src->heads);
    const uint32_t groups = (from->count + group - 1) / group;
    if (groups > 65535) return OKF_E_SHAPE;
    // lengths and weights may be written in place (both kernels say why), not beside their places
    const uint64_t apart = from->len > to->len ? from->len - to->len : to->len - from->len;
    if (apart && apart < from->count) return OKF_E_ARG;
    if (w_out && !(w_out == w_in && w_out_stride == w_in_stride) &&
        rows_meet(w_in, w_in_stride, (uint64_t)from->stride * KV_B, w_out, w_out_stride, keep, rows))
        return OKF_E_ARG;
    if ((st = begin(c))) return st;
    hipLaunchKernelGGL(kv_select_kernel, dim3((uint32_t)rows), dim3(EV_NT), 0, c->stream, seqs_of(from),
                       src->heads, keep, sink, recent, w_in, w_in_stride, w_out, w_out_stride, kept);
    const dim3 grid((keep + KV_B - 1) / KV_B, group * src->heads, groups);
    with_dims(src->dim, [&](auto nd) {
        hipLaunchKernelGGL(kv_gather_kernel<decltype(nd)::value>, grid, dim3(KV_NT), 0, c->stream, cache_of(src), seqs_of(from),
                           cache_of(dst), seqs_of(to), keep, (const int32_t *)kept);
    });
    return finish(c);
}

}  // extern "C"
