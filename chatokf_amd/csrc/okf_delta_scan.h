// okf_delta_scan.h -- the gated delta rule in chunks of 32 tokens on the matrix cores
// (okf_delta_prompt).
//
// With G the running sum of g in a chunk, S the state in front of it and
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),   T = (I + A)^-1 diag(beta),
//   P_ij = e^(G_i - G_j) q_i.k_j (j <= i)
// the chunk's corrections, outputs and the state behind it are
//   U = T (V - e^G K S),   O = scale (e^G Q S + P U),   S' = e^G_last S + K^T (e^(G_last - G) U).
// delta_prepare_kernel computes T and P of every chunk at once and leaves them, with K, Q and K^T, in
// scratch as the operands of the matrix instruction; delta_scan_kernel goes through each
// sequence's chunks one behind the other with the state in registers.
//
// Precision: every product has fp32's.  An fp32 value is three bf16 parts (x = x0 + x1 + x2
// exactly, each the next eight bits), f16 inputs are two, bf16 one; of the products of parts those
// below 2^-24 of the whole are left out.  G and its differences are in 64 bits, so that
// decays far apart keep their ratios.  (I + A)^-1 comes from forward substitution, which
// is as stable as the recurrence; powers of A are not.
//
// Where something is not finite, 0 times it in the places that a mask or the order of tokens
// leaves out would spread it to earlier tokens: a chunk whose corrections or outputs show any goes
// through its tokens again one by one.
#pragma once
#include "okf_delta.h"

namespace okf {

constexpr uint32_t DC = 32;                     // tokens a chunk
constexpr uint32_t DV_BYTES = 12 * 1024 + 256;  // scratch of a chunk and value head: T, P; e^G, e^(G_last - G)

typedef __bf16 bf16x8d __attribute__((ext_vector_type(8)));

template <class T>
__host__ __device__ constexpr int dl_parts() { return sizeof(T) == 4 ? 3 : std::is_same<T, _Float16>::value ? 2 : 1; }
// scratch of a chunk and key head: K, Q and K^T in their parts, 32 dimensions 6 KB
__host__ __device__ constexpr uint32_t dl_kq_bytes(int parts, uint32_t k_dim) { return parts * ((k_dim + 31) / 32) * 6144; }

struct ScanArgs {
    DeltaArgs a;
    uint8_t *work;       // of the chunks c0 .. c1 - 1
    uint64_t per_chunk;  // k_heads * kq + v_heads * DV_BYTES
    uint32_t kq, passes; // passes: pairs of value heads of a key head
    uint32_t c0, c1;
    const float *carry_in;  // the state of the sequence that chunk c0 - 1 belongs to
    float *carry_out;       // that of the one that goes on behind c1
};

__device__ __forceinline__ uint32_t dl_chunks(const StateSeqs &s, uint32_t i) {
    const uint2 r = kv_rows(s.start, i, s.n);
    return (r.y - r.x + DC - 1) / DC;
}
// The chunks of the sequences before sequence `seq`.
__device__ __forceinline__ uint32_t dl_before(const StateSeqs &s, uint32_t seq) {
    uint32_t sum = 0;
    for (uint32_t b = 0; b < seq; b += 64) {
        const uint32_t i = b + (threadIdx.x & 63);
        sum += (uint32_t)__builtin_amdgcn_readlane(lanes_sum(i < seq ? dl_chunks(s, i) : 0), 63);
    }
    return sum;
}

// Eight floats -> NP bf16 parts of each.
template <int NP>
__device__ __forceinline__ void dl_split(const float (&x)[8], bf16x8d (&p)[NP]) {
    u32x4 out[NP];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
        for (int n = 0; n < NP; n++) {
            const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
            out[n][j] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
            if (n < NP - 1) a -= __uint_as_float(ua & 0xFFFF0000u), b -= __uint_as_float(ub & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int n = 0; n < NP; n++) p[n] = __builtin_bit_cast(bf16x8d, out[n]);
}

// d + a b over the parts of both whose product counts.
template <int NA, int NB>
__device__ __forceinline__ floatx4 dl_mma(const bf16x8d (&a)[NA], const bf16x8d (&b)[NB], floatx4 d) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j <= 2) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], d, 0, 0, 0);
    return d;
}

// The operand layout (v_mfma_f32_16x16x32): lane l holds row (A) or column (B) l % 16 and, h = l / 16, of 32
// terms those at 4 h + 0..3 and 16 + 4 h + 0..3; the result's column l % 16 and rows 4 h + 0..3.
// So two results below each other are the B operand of the next product as they lie.

// Two fours of T, as parts.
template <class T, int NP>
__device__ __forceinline__ void dl_operand(const T *lo, const T *hi, bool on_lo, bool on_hi, bf16x8d (&p)[NP]) {
    typedef T vec __attribute__((ext_vector_type(4)));
    vec a, b;
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = b[j] = (T)0.0f;
    if (on_lo) a = *(const vec *)lo;
    if (on_hi) b = *(const vec *)hi;
    if constexpr (NP == 1) {
#pragma unroll
        for (int j = 0; j < 4; j++) p[0][j] = a[j], p[0][4 + j] = b[j];
    } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = to_f32(a[j]), x[4 + j] = to_f32(b[j]);
        dl_split<NP>(x, p);
    }
}

constexpr int DP_NT = 128;
constexpr uint32_t DP_ROW = 36;  // floats from a row of a 32 x 32 matrix in LDS to the next: 16-byte rows on different banks

// A wavefront takes a chunk, a key head and two of its value heads: k k^T and q k^T on the
// matrix cores, then each half of the lanes a value head and each lane a column of its T.
template <class T, int KS>
__global__ __launch_bounds__(DP_NT) void delta_prepare_kernel(const ScanArgs p) {
    constexpr int NP = dl_parts<T>();
    const DeltaArgs &a = p.a;
    __shared__ __align__(16) float mem[DP_NT / 64][4][DC * DP_ROW];
    __shared__ double gam[DP_NT / 64][2][DC];
    __shared__ float bet[DP_NT / 64][2][DC];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, h = lane >> 4;
    const uint32_t w = blockIdx.x * (DP_NT / 64) + wave, pass = w % p.passes, kh = w / p.passes % a.k_heads;
    const uint32_t chunk = p.c0 + w / p.passes / a.k_heads;
    if (chunk >= p.c1) return;
    const SeqItem it = kv_find(chunk, a.s.count, [&](uint32_t s) { return dl_chunks(a.s, s); });
    if (it.seq >= a.s.count) return;
    const uint2 r = kv_rows(a.s.start, it.seq, a.s.n);
    const uint32_t first = r.x + it.at * DC, n = min(r.y - first, DC);
    uint8_t *base = p.work + (uint64_t)(chunk - p.c0) * p.per_chunk;
    bf16x8d *kq = (bf16x8d *)(base + kh * p.kq);
    const T *q = (const T *)a.q + kh * a.k_dim, *k = (const T *)a.k + kh * a.k_dim;
    float *kk = mem[wave][0], *qk = mem[wave][1];
    floatx4 akk[3] = {}, aqk[3] = {};
#pragma unroll 2
    for (int ks = 0; ks < KS; ks++) {
        bf16x8d kp[2][NP], qp[2][NP];
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            const uint32_t row = mt * 16 + m, d = 32 * ks + 4 * h;
            const bool lo = row < n && d < a.k_dim, hi = row < n && d + 16 < a.k_dim;
            const uint64_t at = first + row;
            dl_operand<T, NP>(k + at * a.ks + d, k + at * a.ks + d + 16, lo, hi, kp[mt]);
            dl_operand<T, NP>(q + at * a.qs + d, q + at * a.qs + d + 16, lo, hi, qp[mt]);
            if (pass == 0) {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    kq[((i * 2 + mt) * KS + ks) * 64 + lane] = kp[mt][i];
                    kq[(((NP + i) * 2 + mt) * KS + ks) * 64 + lane] = qp[mt][i];
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 3; t++) {  // (the tile above the diagonal is not used)
            akk[t] = dl_mma(kp[t > 0], kp[t > 1], akk[t]);
            aqk[t] = dl_mma(qp[t > 0], kp[t > 1], aqk[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < 3; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t at = ((t > 0) * 16 + 4 * h + i) * DP_ROW + (t > 1) * 16 + m;
            kk[at] = akk[t][i];
            qk[at] = aqk[t][i];
        }
    if (pass == 0) {  // K^T: rows of dimensions, terms of tokens
        for (uint32_t dt = 0; dt < 2 * KS; dt++) {
            const bool on = dt * 16 < a.k_dim;
            float x[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t row = j / 4 * 16 + 4 * h + j % 4;
                x[j] = on && row < n ? to_f32(k[(uint64_t)(first + row) * a.ks + dt * 16 + m]) : 0.0f;
            }
            bf16x8d part[NP];
            dl_split<NP>(x, part);
#pragma unroll
            for (int i = 0; i < NP; i++) kq[NP * 4 * KS * 64 + (i * 2 * KS + dt) * 64 + lane] = part[i];
        }
    }
    // the value heads' decays
    const uint32_t half = lane >> 5, j = lane & 31, group = a.v_heads / a.k_heads;
    const bool on = pass * 2 + half < group;
    const uint32_t vh = kh * group + pass * 2 + (on ? half : 0);
    double G = 0;
    float beta = 0;
    if (j < n) {
        const double g = (double)a.g[(uint64_t)(first + j) * a.gs + vh] * 1.4426950408889634;
        G = g < -1e5 ? -1e5 : g;  // (2^-1e5 is 0; -inf would leave inf - inf behind it)
        beta = a.beta[(uint64_t)(first + j) * a.bs + vh];
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double up = __shfl_up(G, o, 32);
        if (j >= (uint32_t)o) G += up;
    }
    gam[wave][half][j] = G;
    bet[wave][half][j] = beta;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float *A = mem[wave][2 + half], P[DC];
#pragma unroll
    for (uint32_t i = 0; i < DC; i++) {
        const float e = __builtin_amdgcn_exp2f((float)(gam[wave][half][i] - G));
        A[i * DP_ROW + j] = i > j ? bet[wave][half][i] * (e * kk[i * DP_ROW + j]) : 0.0f;
        P[i] = i >= j ? e * qk[i * DP_ROW + j] : 0.0f;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float t[DC];
#pragma unroll
    for (uint32_t i = 0; i < DC; i++) {
        float s = i == j ? 1.0f : 0.0f;
#pragma unroll
        for (uint32_t l = 0; l < i; l++) s = fmaf(-A[i * DP_ROW + l], t[l], s);
        t[i] = s;
    }
    uint8_t *vb = base + a.k_heads * p.kq;
    float *eg = (float *)(vb + (uint64_t)vh * DV_BYTES + 12 * 1024);
    if (on) {
        eg[j] = __builtin_amdgcn_exp2f((float)G);
        eg[DC + j] = __builtin_amdgcn_exp2f((float)(gam[wave][half][DC - 1] - G));
    }
#pragma unroll
    for (int what = 0; what < 2; what++) {  // T, P: columns of lanes to rows of operands, through LDS
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (uint32_t i = 0; i < DC; i++) A[i * DP_ROW + j] = what ? P[i] : t[i] * beta;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (uint32_t z = 0; z < 2 && pass * 2 + z < group; z++) {
            bf16x8d *to = (bf16x8d *)(vb + (uint64_t)(kh * group + pass * 2 + z) * DV_BYTES) + what * 6 * 64;
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                const float *row = mem[wave][2 + z] + (mt * 16 + m) * DP_ROW + 4 * h;
                const floatx4 lo = *(const floatx4 *)row, hi = *(const floatx4 *)(row + 16);
                const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                bf16x8d part[3];
                dl_split<3>(x, part);
#pragma unroll
                for (int i = 0; i < 3; i++) to[(i * 2 + mt) * 64 + lane] = part[i];
            }
        }
    }
}

// The tokens first .. first + n - 1 one by one: S of a lane in the layout of results (rows dt * 16 + 4 h + i,
// column `col`); outputs where `out`.
template <class T, int KS>
__device__ __forceinline__ void dl_tokens(const DeltaArgs &a, uint32_t kh, uint32_t vh, uint32_t col, uint32_t h, uint32_t first, uint32_t n,
                                          floatx4 (&S)[2 * KS], bool out) {
    const T *q = (const T *)a.q + kh * a.k_dim + 4 * h, *k = (const T *)a.k + kh * a.k_dim + 4 * h;
#pragma unroll 1
    for (uint64_t t = first; t < (uint64_t)first + n; t++) {
        const float e = expf(a.g[t * a.gs + vh]), beta = a.beta[t * a.bs + vh], v = to_f32(((const T *)a.v)[t * a.vs + vh * a.v_dim + col]);
        float kr = 0, qr = 0;
#pragma unroll
        for (int dt = 0; dt < 2 * KS; dt++)
            if (dt * 16 < (int)a.k_dim)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    S[dt][i] = e == 0 ? 0.0f : e * S[dt][i];
                    kr = fmaf(to_f32(k[t * a.ks + dt * 16 + i]), S[dt][i], kr);
                }
        const float u = beta * (v - dl_sum_rows(kr));
#pragma unroll
        for (int dt = 0; dt < 2 * KS; dt++)
            if (dt * 16 < (int)a.k_dim)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    S[dt][i] = fmaf(to_f32(k[t * a.ks + dt * 16 + i]), u, S[dt][i]);
                    qr = fmaf(to_f32(q[t * a.qs + dt * 16 + i]), S[dt][i], qr);
                }
        qr = dl_sum_rows(qr);
        if (out && h == 0) ((T *)a.o)[t * a.os + vh * a.v_dim + col] = (T)(qr * a.scale);
    }
}

constexpr int DN_NT = 256;
// LDS of a pair of wavefronts: the state's parts and the corrections of two chunks
__host__ __device__ constexpr uint32_t dl_hand(int KS) { return 3 * KS * 1024 + 2048 + 16; }
template <int KS>
constexpr uint32_t dl_scan_lds() { return 2 * 2 * dl_hand(KS); }

__device__ __forceinline__ void dl_meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A workgroup takes 32 columns of a value head's state through its sequence's chunks, two wavefronts 16 of
// them: the first carries the state from chunk to chunk (K S, U, S'), the second makes the outputs of the chunk
// before from the state's parts and the corrections that the first leaves in LDS.
template <class T, int KS>
__global__ __launch_bounds__(DN_NT, KS * dl_parts<T>() <= 6 ? 2 : 1) void delta_scan_kernel(const ScanArgs p) {
    constexpr int NP = dl_parts<T>();
    const DeltaArgs &a = p.a;
    extern __shared__ __align__(16) uint8_t dn_mem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, h = lane >> 4;
    const uint32_t tiles = a.v_dim / 16, pairs = (tiles + 1) / 2, group = a.v_heads / a.k_heads;
    // a key head's workgroups on one XCD, whose L2 then holds its K and Q (XCDs take workgroups in turn)
    uint32_t id = blockIdx.x;
    const uint32_t each = group * pairs, sets = a.s.count * a.k_heads;
    if (sets % 8 == 0) id = (id / 8 / each * 8 + id % 8) * each + id / 8 % each;
    const uint32_t tile = id % pairs * 2 + (wave >> 1), vh = id / pairs % a.v_heads, seq = id / pairs / a.v_heads, kh = vh / group;
    const uint2 r = kv_rows(a.s.start, seq, a.s.n);
    const uint32_t own = (r.y - r.x + DC - 1) / DC, c_own = dl_before(a.s, seq);
    const uint32_t cb = max(c_own, p.c0), ce = min(c_own + own, p.c1);
    const bool begins = !own || c_own >= p.c0, ends = !own || c_own + own <= p.c1;
    if (own ? cb >= ce : p.c0 != 0) return;
    const uint32_t n = own ? ce - cb : 0;
    if (tile >= tiles) {  // (an odd number of column tiles)
        for (uint32_t c = 0; c < n; c++) dl_meet();
        return;
    }
    const uint32_t col = tile * 16 + m, row0 = r.x + (cb - c_own) * DC;  // (n: row0 is not used without chunks)
    uint8_t *hand = dn_mem + (wave >> 1) * 2 * dl_hand(KS);
    const uint8_t *work = p.work + (uint64_t)(cb - p.c0) * p.per_chunk;
    auto kq_of = [&](uint32_t c) { return (const bf16x8d *)(work + c * p.per_chunk + kh * p.kq) + lane; };
    auto vb_of = [&](uint32_t c) { return work + c * p.per_chunk + a.k_heads * p.kq + (uint64_t)vh * DV_BYTES; };
    const int64_t slot = a.s.state(seq);
    if ((wave & 1) == 0) {
        floatx4 S[2 * KS];
        const uint64_t each_state = (uint64_t)a.v_heads * a.k_dim * a.v_dim, at = ((uint64_t)vh * a.k_dim + 4 * h) * a.v_dim + col;
        const float *from = !begins ? p.carry_in : a.si && slot >= 0 ? a.si + slot * each_state : nullptr;
#pragma unroll
        for (int dt = 0; dt < 2 * KS; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[dt][i] = from && dt * 16 < (int)a.k_dim ? from[at + (uint64_t)(dt * 16 + i) * a.v_dim] : 0.0f;
        bf16x8d ka[2][KS][NP], tp[2][3], kt[2 * KS][NP];
        T vv[8];
        floatx4 eg[2], el[2];
        float e_last;
        auto load_k = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int i = 0; i < NP; i++) ka[mt][ks][i] = kq[((i * 2 + mt) * KS + ks) * 64];
        };
        auto load_v = [&](uint32_t c) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t row = row0 + c * DC + j / 4 * 16 + 4 * h + j % 4;
                vv[j] = ((const T *)a.v)[(uint64_t)min(row, r.y - 1) * a.vs + vh * a.v_dim + col];
            }
            const floatx4 *e = (const floatx4 *)(vb_of(c) + 12 * 1024) + h;
            eg[0] = e[0], eg[1] = e[4];
        };
        auto load_t = [&](uint32_t c) {
            const bf16x8d *to = (const bf16x8d *)vb_of(c) + lane;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 3; i++) tp[mt][i] = to[(i * 2 + mt) * 64];
        };
        auto load_kt = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c) + NP * 4 * KS * 64;
#pragma unroll
            for (int dt = 0; dt < 2 * KS; dt++)
#pragma unroll
                for (int i = 0; i < NP; i++) kt[dt][i] = kq[(i * 2 * KS + dt) * 64];
            const float *e = (const float *)(vb_of(c) + 12 * 1024);
            el[0] = ((const floatx4 *)(e + DC))[h], el[1] = ((const floatx4 *)(e + DC))[4 + h];
            e_last = e[DC - 1];
        };
        if (n) load_k(0), load_v(0), load_t(0), load_kt(0);
        for (uint32_t c = 0; c < n; c++) {
            const uint32_t next = min(c + 1, n - 1), first = row0 + c * DC, left = r.y - first;
            bf16x8d *sp = (bf16x8d *)(hand + (c & 1) * dl_hand(KS)) + lane;
            floatx4 ks0[2] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float x[8] = {S[2 * ks][0],     S[2 * ks][1],     S[2 * ks][2],     S[2 * ks][3],
                                    S[2 * ks + 1][0], S[2 * ks + 1][1], S[2 * ks + 1][2], S[2 * ks + 1][3]};
                bf16x8d part[3];
                dl_split<3>(x, part);
#pragma unroll
                for (int i = 0; i < 3; i++) sp[(ks * 3 + i) * 64] = part[i];
#pragma unroll
                for (int mt = 0; mt < 2; mt++) ks0[mt] = dl_mma(ka[mt][ks], part, ks0[mt]);
            }
            load_k(next);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = (uint32_t)(j / 4 * 16 + 4 * h + j % 4) < left ? to_f32(vv[j]) : 0.0f;
                x[j] = v - eg[j / 4][j % 4] * ks0[j / 4][j % 4];
            }
            load_v(next);
            bf16x8d part[3];
            dl_split<3>(x, part);
            floatx4 u[2];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) u[mt] = dl_mma(tp[mt], part, floatx4{0, 0, 0, 0});
#pragma unroll
            for (int dt = 0; dt < 2 * KS; dt++) S[dt] *= e_last;
            load_t(next);
            floatx4 *up = (floatx4 *)(sp - lane + 3 * KS * 64) + lane;
            up[0] = u[0];
            up[64] = u[1];
            float bad = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                bad = fmaf(u[j / 4][j % 4], 0.0f, bad);
                x[j] = el[j / 4][j % 4] * u[j / 4][j % 4];
            }
            const bool careful = __ballot(bad != bad) != 0;
            if (lane == 0) *(uint32_t *)(up - lane + 128) = careful;
            if (careful) {
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const bf16x8d p0 = sp[(ks * 3) * 64], p1 = sp[(ks * 3 + 1) * 64], p2 = sp[(ks * 3 + 2) * 64];
#pragma unroll
                    for (int j = 0; j < 8; j++) S[2 * ks + j / 4][j % 4] = ((float)p0[j] + (float)p1[j]) + (float)p2[j];
                }
                dl_tokens<T, KS>(a, kh, vh, col, h, first, min(left, DC), S, true);
            } else {
                dl_split<3>(x, part);
#pragma unroll
                for (int dt = 0; dt < 2 * KS; dt++) S[dt] = dl_mma(kt[dt], part, S[dt]);
            }
            load_kt(next);
            dl_meet();
        }
        float *to = !ends ? p.carry_out : a.so && slot >= 0 ? a.so + slot * each_state : nullptr;
        if (to) {
#pragma unroll
            for (int dt = 0; dt < 2 * KS; dt++)
                if (dt * 16 < (int)a.k_dim)
#pragma unroll
                    for (int i = 0; i < 4; i++) to[at + (uint64_t)(dt * 16 + i) * a.v_dim] = S[dt][i];
        }
    } else {
        bf16x8d qa[2][KS][NP], pp[2][3];
        floatx4 eg[2];
        auto load_q = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c) + NP * 2 * KS * 64;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int i = 0; i < NP; i++) qa[mt][ks][i] = kq[((i * 2 + mt) * KS + ks) * 64];
        };
        auto load_p = [&](uint32_t c) {
            const bf16x8d *to = (const bf16x8d *)vb_of(c) + 6 * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 3; i++) pp[mt][i] = to[(i * 2 + mt) * 64];
            const floatx4 *e = (const floatx4 *)(vb_of(c) + 12 * 1024) + h;
            eg[0] = e[0], eg[1] = e[4];
        };
        if (n) load_q(0), load_p(0);
        for (uint32_t c = 0; c < n; c++) {
            dl_meet();
            const uint32_t next = min(c + 1, n - 1), first = row0 + c * DC, left = r.y - first;
            const bf16x8d *sp = (const bf16x8d *)(hand + (c & 1) * dl_hand(KS)) + lane;
            floatx4 o[2] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                bf16x8d part[3];
#pragma unroll
                for (int i = 0; i < 3; i++) part[i] = sp[(ks * 3 + i) * 64];
#pragma unroll
                for (int mt = 0; mt < 2; mt++) o[mt] = dl_mma(qa[mt][ks], part, o[mt]);
            }
            load_q(next);
            const floatx4 *up = (const floatx4 *)(sp - lane + 3 * KS * 64) + lane;
            const floatx4 u0 = up[0], u1 = up[64];
            const bool done = *(const uint32_t *)(up - lane + 128);
            const float x[8] = {u0[0], u0[1], u0[2], u0[3], u1[0], u1[1], u1[2], u1[3]};
            bf16x8d part[3];
            dl_split<3>(x, part);
            float bad = 0;
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                o[mt] = dl_mma(pp[mt], part, o[mt] * eg[mt]);
#pragma unroll
                for (int i = 0; i < 4; i++) bad = fmaf(o[mt][i], 0.0f, bad);
            }
            load_p(next);
            if (done) continue;
            if (__ballot(bad != bad)) {
                floatx4 S[2 * KS];
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const bf16x8d p0 = sp[(ks * 3) * 64], p1 = sp[(ks * 3 + 1) * 64], p2 = sp[(ks * 3 + 2) * 64];
#pragma unroll
                    for (int j = 0; j < 8; j++) S[2 * ks + j / 4][j % 4] = ((float)p0[j] + (float)p1[j]) + (float)p2[j];
                }
                dl_tokens<T, KS>(a, kh, vh, col, h, first, min(left, DC), S, true);
                continue;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t row = j / 4 * 16 + 4 * h + j % 4;
                if (row < left) ((T *)a.o)[(uint64_t)(first + row) * a.os + vh * a.v_dim + col] = (T)(o[j / 4][j % 4] * a.scale);
            }
        }
    }
}

}  // namespace okf
