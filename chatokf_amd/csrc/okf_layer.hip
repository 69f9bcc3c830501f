// okf_layer.hip -- the C ABI of what stands around the projections (include/okf_quant.h):
// head norms with rotation, the short convolution and the gated delta rule, over
// okf_rope.h, okf_conv.h and okf_delta.h.
#include "okf_impl.h"
#include "okf_args.h"
#include "okf_rope.h"
#include "okf_delta_run.h"

#include <cmath>

namespace {

using namespace okf;
using namespace okf_impl;

constexpr uint32_t ROWS_MAX = 0x7FFFFF00u;  // (rows are counted in 32 bits with a sign, up to a workgroup's past the last)

// The frequencies of okf_rope in turns a position, 64 bits: base^(-2 i / rot) as a product of
// two powers, so that no error grows with i.
int rope_freqs(const okf_rope &r, double *f, float &mag) {
    mag = r.mag;
    if (!r.rot) return OKF_OK;
    if (!(r.base > 0) || !std::isfinite(r.base) || !(r.factor > 0) || !std::isfinite(r.factor) || !std::isfinite(r.mag)) return OKF_E_ARG;
    const uint32_t n = r.rot / 2;
    double low = 0, width = 1;
    if (r.original) {
        if (!(r.base > 1) || !(r.beta_fast > 0) || !(r.beta_slow > 0) || !std::isfinite(r.beta_fast) || !std::isfinite(r.beta_slow)) return OKF_E_ARG;
        auto at = [&](double turns) { return r.rot * std::log(r.original / (turns * 2 * M_PI)) / (2 * std::log((double)r.base)); };
        low = std::max(std::floor(at(r.beta_fast)), 0.0);
        width = std::max(std::min(std::ceil(at(r.beta_slow)), r.rot - 1.0) - low, 0.001);
        if (!mag) mag = r.factor > 1 ? (float)(0.1 * std::log((double)r.factor) + 1) : 1.0f;
    }
    if (!mag) mag = 1.0f;
    double high[16], few[8];
    for (uint32_t j = 0; j < 16 && 8 * j < n; j++) high[j] = std::pow((double)r.base, -16.0 * j / r.rot);
    for (uint32_t j = 0; j < 8; j++) few[j] = std::pow((double)r.base, -2.0 * j / r.rot);
    for (uint32_t i = 0; i < n; i++) {
        const double ramp = r.original ? std::min(std::max((i - low) / width, 0.0), 1.0) : 1.0;
        f[i] = high[i / 8] * few[i % 8] * (ramp / r.factor + 1 - ramp) / (2 * M_PI);
    }
    return OKF_OK;
}

// Bytes of a row whose heads stand `head` values apart.
uint64_t row_bytes(uint32_t heads, uint64_t head, uint32_t dim, uint32_t size) { return ((heads - 1) * head + dim) * size; }

// Whether two heads of n rows, `row` values apart, of `heads` heads, `head` apart, share any of their dim values.  Rows
// of one head do not (row >= dim), nor heads of one row; head h of a row starts h * head behind the row's first
// head, and of those only the nearest two, one on either side, can be less than dim away.
bool heads_meet(uint64_t row, uint64_t head, uint32_t n, uint32_t heads, uint32_t dim) {
    if (row >= (heads - 1) * head + dim || head >= (unsigned __int128)(n - 1) * row + dim) return false;
    for (uint32_t h = 1; h < heads; h++) {
        const uint64_t r = h * head / row, past = h * head % row;
        if ((r < n && past < dim) || (r + 1 < n && row - past < dim)) return true;
    }
    return false;
}

template <class T, int L>
void launch_rope(okf_ctx *c, const RopeArgs &a, bool cross, uint32_t grid) {
    if (cross) hipLaunchKernelGGL((norm_rope_kernel<T, L, true>), dim3(grid), dim3(RP_NT), 0, c->stream, a);
    else hipLaunchKernelGGL((norm_rope_kernel<T, L, false>), dim3(grid), dim3(RP_NT), 0, c->stream, a);
}

template <class T, int W>
void launch_conv(okf_ctx *c, const ConvArgs &a, bool wide, dim3 grid) {
    constexpr int V = 16 / sizeof(T);
    if (wide) hipLaunchKernelGGL((conv_kernel<T, W, V>), grid, dim3(256), 0, c->stream, a);
    else hipLaunchKernelGGL((conv_kernel<T, W, 1>), grid, dim3(256), 0, c->stream, a);
}

int check_states(const okf_state_seqs *s) {
    if (!s || !s->start) return OKF_E_ARG;
    if (!s->seqs || !s->n || s->n > ROWS_MAX || s->seqs > ROWS_MAX || !s->slots || s->slots > ROWS_MAX) return OKF_E_SHAPE;
    if (!s->slot && s->slots < s->seqs) return OKF_E_SHAPE;
    if (!aligned4(s->start) || !aligned4(s->slot)) return OKF_E_SHAPE;
    return OKF_OK;
}

// `each` bytes a state: in place, or apart.
bool states_apart(const okf_state_seqs *s, uint64_t each) {
    if (!s->state_in || !s->state_out || s->state_in == s->state_out) return true;
    return rows_apart(s->state_in, each, each, s->slots, s->state_out, each, each, s->slots);
}

// Whether states of `each` bytes share no memory with n rows of `row` bytes that the call reads or writes.
bool state_apart(const void *state, const okf_state_seqs *s, uint64_t each, const void *p, uint64_t stride, uint64_t row) {
    return !state || rows_apart(state, each, each, s->slots, p, stride, row, s->n);
}

StateSeqs seqs_of(const okf_state_seqs *s) { return {s->start, s->slot, s->seqs, s->n, s->slots}; }

int check_delta(const okf_delta *d, const okf_state_seqs *s, DeltaArgs &a, bool over_v) {
    if (!d || !d->q || !d->k || !d->v || !d->g || !d->beta || !d->o) return OKF_E_ARG;
    int st = check_states(s);
    if (st) return st;
    if (!attn_type(d->type)) return OKF_E_TYPE;
    if (!d->k_heads || !d->v_heads || d->v_heads % d->k_heads || d->v_heads > 65535 || !good_dim(d->k_dim) || !good_dim(d->v_dim)) return OKF_E_SHAPE;
    const uint32_t size = d->type == F32 ? 4 : 2, kw = d->k_heads * d->k_dim, vw = d->v_heads * d->v_dim;
    a = DeltaArgs{d->q, d->k, d->v, d->g, d->beta, d->o, d->q_stride, d->k_stride, d->v_stride, d->o_stride, d->g_stride, d->beta_stride,
                  d->k_heads, d->v_heads, d->k_dim, d->v_dim, d->scale, (const float *)s->state_in, (float *)s->state_out, seqs_of(s)};
    if (!row_stride(a.qs, kw, size) || !row_stride(a.ks, kw, size) || !row_stride(a.vs, vw, size) || !row_stride(a.os, vw, size)) return OKF_E_SHAPE;
    for (uint64_t *g : {&a.gs, &a.bs}) {
        if (!*g) *g = d->v_heads;
        if (*g < d->v_heads || *g > 1ull << 40) return OKF_E_SHAPE;
    }
    if (!aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->o) || !aligned4(d->g) || !aligned4(d->beta) ||
        !aligned16(s->state_in) || !aligned16(s->state_out))
        return OKF_E_SHAPE;
    const uint64_t each = (uint64_t)d->v_heads * d->k_dim * d->v_dim * sizeof(float);
    if (!states_apart(s, each)) return OKF_E_ARG;
    auto apart = [&](const void *p, uint64_t stride, uint64_t row) {
        return rows_apart(d->o, a.os * size, vw * size, s->n, p, stride, row, s->n);
    };
    if (!apart(d->q, a.qs * size, kw * size) || !apart(d->k, a.ks * size, kw * size) || !apart(d->g, a.gs * 4, d->v_heads * 4) ||
        !apart(d->beta, a.bs * 4, d->v_heads * 4))
        return OKF_E_ARG;
    if (!(over_v && d->o == d->v && a.os == a.vs) && !apart(d->v, a.vs * size, vw * size)) return OKF_E_ARG;
    auto kept_apart = [&](const void *p, uint64_t stride, uint64_t row) { return state_apart(s->state_out, s, each, p, stride, row); };
    if (!kept_apart(d->o, a.os * size, vw * size) || !state_apart(s->state_in, s, each, d->o, a.os * size, vw * size) ||
        !kept_apart(d->q, a.qs * size, kw * size) || !kept_apart(d->k, a.ks * size, kw * size) || !kept_apart(d->v, a.vs * size, vw * size) ||
        !kept_apart(d->g, a.gs * 4, d->v_heads * 4) || !kept_apart(d->beta, a.bs * 4, d->v_heads * 4))
        return OKF_E_ARG;
    // (grids of less than 2^32 threads)
    if ((uint64_t)s->seqs * d->v_heads * (d->v_dim / 16) > 0x3FFFFFFull - 8) return OKF_E_SHAPE;
    return OKF_OK;
}

int run_step(okf_ctx *c, int32_t type, const DeltaArgs &a) {
    with_type(type, [&](auto t) { launch_delta_step<decltype(t)>(c, a); });
    return finish(c);
}

// The chunks of okf_delta_prompt: how many there may be, how many at a time (their scratch in
// DELTA_WORK bytes, a grid of less than 2^32 threads), and the bytes of a chunk and of two states
// that go from one launch to the next.
constexpr uint64_t DELTA_WORK = 512ull << 20;
// Prompts of no more rows go token by token.  One sequence's 16 tokens by steps, and 17 in chunks (us): 48 heads of 128 x 128
// 20.9 and 22 fp32, 15.9 and 17 bf16; 24 of 96 x 208 bf16 14.0 and 15.1; 4 of 64 x 64 fp32 11.7 and 14.7; 32 of 256 x 256 21.3 and
// 37 fp32, 22.2 and 25.1 bf16.  (The call's rows are counted: 8 sequences of 4 fp32 tokens, 48 heads, take 67 in chunks and
// 12.8 by okf_delta_step, which is for such calls.)
constexpr uint32_t DELTA_FEW = 16;
struct DeltaPlan {
    uint64_t chunks, at_once, per_chunk, carry;
    uint32_t kq, passes;
    DeltaPlan(int32_t type, uint32_t n, uint32_t seqs, uint32_t k_heads, uint32_t v_heads, uint32_t k_dim, uint32_t v_dim) {
        kq = dl_kq_bytes(type == F32 ? 3 : type == F16 ? 2 : 1, k_dim);
        passes = (v_heads / k_heads + 1) / 2;
        per_chunk = (uint64_t)k_heads * kq + (uint64_t)v_heads * DV_BYTES;
        carry = 2ull * v_heads * k_dim * v_dim * sizeof(float);
        chunks = std::min<uint64_t>(n, n / DC + (uint64_t)seqs);
        at_once = std::min<uint64_t>(std::max<uint64_t>(DELTA_WORK / per_chunk, 1), (1u << 24) / (k_heads * passes));
        at_once = std::min(std::max<uint64_t>(at_once, 1), chunks);
    }
    uint64_t bytes(uint64_t n) const { return carry + n * per_chunk; }
};

int run_prompt(okf_ctx *c, int32_t type, const DeltaArgs &a) {
    DeltaPlan pl(type, a.s.n, a.s.count, a.k_heads, a.v_heads, a.k_dim, a.v_dim);
    const uint64_t blocks = (uint64_t)a.s.count * a.v_heads * ((a.v_dim / 16 + 1) / 2);
    if (a.s.n <= DELTA_FEW || blocks > 0xFFFFFFull) return run_step(c, type, a);
    const uint64_t least = std::min<uint64_t>(pl.at_once, 16);
    uint64_t n = pl.at_once;
    while (pl.bytes(n) > c->part_bytes && grow_part(c, pl.bytes(n), true) != OKF_OK) {  // (what there is, or a quarter as much)
        const uint64_t fit = c->part_bytes > pl.carry ? (c->part_bytes - pl.carry) / pl.per_chunk : 0;
        if (fit < least && n / 4 < least) return run_step(c, type, a);
        n = fit < least ? n / 4 : std::min(fit, n);
    }
    note_capture(c, false, true, false);
    float *carry = c->part;
    const uint64_t state = pl.carry / 2 / sizeof(float);
    uint8_t *work = (uint8_t *)(carry + 2 * state);
    ScanArgs p{a, work, work + n * a.k_heads * pl.kq, pl.kq, pl.passes, 0, 0, (uint32_t)n, carry, carry + state};
    for (uint64_t at = 0; at < pl.chunks; at += n) {
        p.c0 = (uint32_t)at, p.c1 = (uint32_t)std::min(at + n, pl.chunks);
        with_type(type, [&](auto t) { launch_delta_chunks<decltype(t)>(c, p); });
        const float *out = p.carry_out;
        p.carry_out = (float *)p.carry_in;
        p.carry_in = out;
    }
    return finish(c);
}

}  // namespace

extern "C" {

int okf_norm_rope_rows(okf_ctx *c, const okf_norm_rope *p) {
    if (!p || !p->q || !p->q_out || !p->k != !p->k_out || (p->rope.rot && !p->pos)) return OKF_E_ARG;
    if (!attn_type(p->type)) return OKF_E_TYPE;
    const okf_rope &r = p->rope;
    if (!p->heads || p->heads > 65535 || (p->k && (!p->kv_heads || p->kv_heads > 65535)) || !good_dim(p->dim) || !p->n || p->n > ROWS_MAX ||
        r.rot % 2 || r.rot > p->dim)
        return OKF_E_SHAPE;
    const uint32_t size = p->type == F32 ? 4 : 2, kv = p->k ? p->kv_heads : 0, V = 16 / size;
    RopeArgs a{p->q, p->k, p->q_out, p->k_out, p->q_stride, p->k_stride, p->q_out_stride, p->k_out_stride, p->q_head, p->k_head,
               p->q_out_head, p->k_out_head, p->q_norm, p->k_norm, r.rot ? r.div : nullptr, p->pos, p->heads, kv, p->dim, p->n, r.rot, r.pairs,
               0, 0, 0, 0, p->eps, 1.0f, {}};
    // (rows may lie inside a head's plane, heads inside a row: either stride may be the larger)
    for (uint64_t *s : {&a.qs, &a.qos})
        if (!*s) *s = (uint64_t)p->heads * p->dim;
    for (uint64_t *s : {&a.ks, &a.kos})
        if (!*s) *s = (uint64_t)std::max(kv, 1u) * p->dim;
    for (uint64_t *s : {&a.qs, &a.ks, &a.qos, &a.kos, &a.qh, &a.kh, &a.qoh, &a.koh})
        if (!row_stride(*s, p->dim, size)) return OKF_E_SHAPE;
    if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->q_out) || !aligned16(p->k_out) || !aligned4(p->q_norm) || !aligned4(p->k_norm) ||
        !aligned4(p->pos) || !aligned4(a.div))
        return OKF_E_SHAPE;
    struct Rows {
        const void *p;
        uint64_t stride, head;
        uint32_t heads;
    };
    const Rows q{p->q, a.qs, a.qh, p->heads}, k{p->k, a.ks, a.kh, kv}, qo{p->q_out, a.qos, a.qoh, p->heads}, ko{p->k_out, a.kos, a.koh, kv};
    auto apart = [&](const Rows &x, const Rows &y) {
        return !x.p || !y.p || rows_apart(x.p, x.stride * size, row_bytes(x.heads, x.head, p->dim, size), p->n, y.p, y.stride * size,
                                          row_bytes(y.heads, y.head, p->dim, size), p->n);
    };
    auto same = [](const Rows &x, const Rows &y) { return x.p == y.p && x.stride == y.stride && x.head == y.head; };
    if ((!same(q, qo) && !apart(q, qo)) || (!same(k, ko) && !apart(k, ko)) || !apart(q, ko) || !apart(k, qo) || !apart(qo, ko)) return OKF_E_ARG;
    if (heads_meet(a.qos, a.qoh, p->n, p->heads, p->dim) || (kv && heads_meet(a.kos, a.koh, p->n, kv, p->dim))) return OKF_E_ARG;
    int st = rope_freqs(r, a.f, a.mag);
    if (st) return st;
    if ((st = begin(c))) return st;
    // lanes a head: 32 bytes each, a power of two
    uint32_t L = 1;
    while (L * 2 * V < p->dim) L *= 2;
    const uint32_t G = 64 / L;
    a.tq = (p->heads + G - 1) / G;
    a.tk = (kv + G - 1) / G;
    const uint32_t tasks = a.tq + a.tk;
    // tasks a wavefront: as many as leave 32 wavefronts a CU (4943 rows of 16 + 4 f16 heads of 256: 27.5 us, with 16 or 64
    // wavefronts 29.6 and 32.8; 8192 rows of 40 + 8 bf16 heads of 128 43.3, 43.2 and 44.5)
    a.per = std::max(1u, (uint32_t)std::min<uint64_t>(tasks, (uint64_t)p->n * tasks / (32 * c->cus)));
    a.wpr = (tasks + a.per - 1) / a.per;
    // (a grid of less than 2^32 threads; where rows are left a wavefront takes the next)
    const uint64_t waves = std::min<uint64_t>((uint64_t)p->n * a.wpr, (uint64_t)((1u << 22) / a.wpr + 1) * a.wpr);
    uint64_t grid = (waves + RP_NT / 64 - 1) / (RP_NT / 64);
    while (grid * (RP_NT / 64) % a.wpr) grid++;
    const bool cross = !r.pairs && r.rot / 2 % V;
    with_type(p->type, [&](auto t) {
        using T = decltype(t);
        switch (L) {
        case 1: launch_rope<T, 1>(c, a, cross, (uint32_t)grid); break;
        case 2: launch_rope<T, 2>(c, a, cross, (uint32_t)grid); break;
        case 4: launch_rope<T, 4>(c, a, cross, (uint32_t)grid); break;
        case 8: launch_rope<T, 8>(c, a, cross, (uint32_t)grid); break;
        case 16: launch_rope<T, 16>(c, a, cross, (uint32_t)grid); break;
        default: launch_rope<T, 32>(c, a, cross, (uint32_t)grid); break;
        }
    });
    return finish(c);
}

int okf_conv_rows(okf_ctx *c, const okf_conv *p, const okf_state_seqs *s) {
    if (!p || !p->x || !p->y || !p->w) return OKF_E_ARG;
    int st = check_states(s);
    if (st) return st;
    if (!attn_type(p->type)) return OKF_E_TYPE;
    if (!p->channels || p->width < 2 || p->width > 8) return OKF_E_SHAPE;
    const uint32_t size = p->type == F32 ? 4 : 2, V = 16 / size;
    ConvArgs a{p->x, s->state_in, p->y, s->state_out, p->w, p->bias, p->x_stride, p->y_stride, p->channels, (uint32_t)(p->silu != 0), 0, seqs_of(s)};
    for (uint64_t *r : {&a.xs, &a.ys}) {
        if (!*r) *r = p->channels;
        if (*r < p->channels || *r > 1ull << 40) return OKF_E_SHAPE;
    }
    if (((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)s->state_in | (uintptr_t)s->state_out) & (size - 1) || !aligned4(p->w) || !aligned4(p->bias))
        return OKF_E_SHAPE;
    // 16-byte pieces where every row begins and ends with a whole one
    const bool wide = p->channels % V == 0 && a.xs % V == 0 && a.ys % V == 0 && aligned16(p->x) && aligned16(p->y) && aligned16(s->state_in) &&
                      aligned16(s->state_out);
    const uint64_t per = 256ull * (wide ? V : 1), gy = (p->channels + per - 1) / per;
    // rows a thread, in whole groups of 8 up to 32: more than 8 only where that leaves more than one workgroup a CU, two just
    // before each step (10240 bf16 channels: 64 rows 7.5 us by 8 and 13.6 by 32, 2000 21.9 and 23.5, by 24 20.3, 16000 162
    // and 142, by 64 145)
    const uint64_t few = 16ull * (c ? c->cus : 256);
    a.rows = (uint32_t)std::min<uint64_t>((s->n * gy + few - 1) / few, 4) * 8;
    auto count = [&] { return std::min<uint64_t>(s->n, s->n / a.rows + s->seqs) + s->seqs; };
    while (count() * gy > 0xFFFFFFull && a.rows < 1u << 16) a.rows *= 2;
    const uint64_t items = count();
    if (gy > 65535 || items * gy > 0xFFFFFFull) return OKF_E_SHAPE;  // (a grid of less than 2^32 threads)
    if (!rows_apart(p->x, a.xs * size, (uint64_t)p->channels * size, s->n, p->y, a.ys * size, (uint64_t)p->channels * size, s->n)) return OKF_E_ARG;
    const uint64_t each = (uint64_t)(p->width - 1) * p->channels * size, row = (uint64_t)p->channels * size;
    if (!states_apart(s, each) || !state_apart(s->state_out, s, each, p->x, a.xs * size, row) ||
        !state_apart(s->state_out, s, each, p->y, a.ys * size, row) || !state_apart(s->state_in, s, each, p->y, a.ys * size, row))
        return OKF_E_ARG;
    if ((st = begin(c))) return st;
    const dim3 grid((uint32_t)items, (uint32_t)gy);
    with_type(p->type, [&](auto t) {
        using T = decltype(t);
        switch (p->width) {
        case 2: launch_conv<T, 2>(c, a, wide, grid); break;
        case 3: launch_conv<T, 3>(c, a, wide, grid); break;
        case 4: launch_conv<T, 4>(c, a, wide, grid); break;
        case 5: launch_conv<T, 5>(c, a, wide, grid); break;
        case 6: launch_conv<T, 6>(c, a, wide, grid); break;
        case 7: launch_conv<T, 7>(c, a, wide, grid); break;
        default: launch_conv<T, 8>(c, a, wide, grid); break;
        }
    });
    return finish(c);
}

int okf_delta_step(okf_ctx *c, const okf_delta *d, const okf_state_seqs *s) {
    DeltaArgs a;
    int st = check_delta(d, s, a, true);
    if (st) return st;
    if ((st = begin(c))) return st;
    return run_step(c, d->type, a);
}

int okf_delta_prompt(okf_ctx *c, const okf_delta *d, const okf_state_seqs *s) {
    DeltaArgs a;
    int st = check_delta(d, s, a, false);
    if (st) return st;
    if ((st = begin(c))) return st;
    return run_prompt(c, d->type, a);
}

int okf_delta_reserve(okf_ctx *c, int32_t type, uint32_t n, uint32_t seqs, uint32_t k_heads, uint32_t v_heads, uint32_t k_dim,
                      uint32_t v_dim) {
    if (!c) return OKF_E_ARG;
    if (!attn_type(type)) return OKF_E_TYPE;
    if (!n || n > ROWS_MAX || !seqs || seqs > ROWS_MAX || !k_heads || !v_heads || v_heads % k_heads || v_heads > 65535 || !good_dim(k_dim) ||
        !good_dim(v_dim))
        return OKF_E_SHAPE;
    if (c->device < 0) return OKF_E_NODEV;
    (void)hipSetDevice(c->device);
    const DeltaPlan pl(type, n, seqs, k_heads, v_heads, k_dim, v_dim);
    const bool reserved = c->reserved;
    c->reserved = false;
    const int st = grow_part(c, pl.bytes(pl.at_once));
    c->reserved = reserved;
    return st;
}

}  // extern "C"
