// Attention over the paged key/value cache (include/q3c.h, q3c_kv_attend): causal by position, optional sliding window with first
// tokens that stay visible, grouped heads, f32 / bf16 / 4-bit pages, any number of new tokens per request.
#include "kv.h"

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// What one tile of 16 query columns works on.  The new tokens of a request and the heads that share a kv head make its columns: column
// c is token c / group, head c % group of the kv head, so one new token of a grouped model fills part of one tile and a prompt many.
// Tiles of all requests are numbered through: request b's start at offsets[b] * group / 16 + b, which leaves room for its
// rounded-up last one, so the grid needs only the totals that the host knows.
struct Tile {
    int seq, row, tok0, ncols, col0;    // request, table row (-1: bad), its first token, columns in all, first column of the tile
    int first_pos;                      // position of its first new token
    int pmin, pmax;                     // positions that exist among the tile's columns (pmax < pmin: none)
    bool on;
};
__device__ __forceinline__ Tile kv_tile(const KvAttendArgs& a, int x, int cols, int lane) {
    Tile t;
    const int S = a.b.sequences, G = a.group;
    int n = 1;
    t.on = false;
    if (a.b.offsets) {
        int b = 0;
        for (int i = 0; i < S; i += 64) {
            const int j = min(i + lane, S - 1) + 1;
            const int o = min(max(a.b.offsets[j], 0), a.b.tokens);
            b += __popcll(__ballot(i + lane < S && (int)((long long)o * G / cols) + j <= x));
        }
        if (b >= S) return t;
        t.tok0 = min(max(a.b.offsets[b], 0), a.b.tokens);
        n = min(max(a.b.offsets[b + 1], 0), a.b.tokens) - t.tok0;
        t.seq = b;
        t.col0 = (x - ((int)((long long)t.tok0 * G / cols) + b)) * cols;
    } else {
        const int per = (G + cols - 1) / cols;
        t.seq = t.tok0 = x / per;
        if (t.seq >= S) return t;
        t.col0 = (x - t.seq * per) * cols;
    }
    if (n < 1 || t.col0 < 0 || t.col0 >= (long long)n * G) return t;
    t.ncols = n * G;
    t.on = true;
    const int row = a.b.rows[t.seq];
    t.row = row >= 0 && row < a.c.rows ? row : -1;
    t.pmin = 0;
    t.pmax = -1;
    if (t.row < 0) return t;
    t.first_pos = a.c.lens[row] - n;
    const int i0 = t.col0 / G, i1 = min(t.col0 + cols, t.ncols) - 1;
    t.pmin = max(t.first_pos + i0, 0);
    t.pmax = min(t.first_pos + i1 / G, (a.c.width << a.c.ps_shift) - 1);
    return t;
}
// The keys a tile can see, in aligned chunks of TB tokens: the first `sinks` tokens' chunks, then from the window's start to the end.
struct Span {
    int sink_chunks, first, total;
    __device__ __forceinline__ int chunk(int i) const { return i < sink_chunks ? i : first + i - sink_chunks; }
};
__device__ __forceinline__ Span kv_span(const KvAttendArgs& a, const Tile& t, int tb) {
    Span s;
    s.sink_chunks = s.first = s.total = 0;
    if (t.pmax < t.pmin) return s;
    int lo = 0;
    if (a.window > 0) {
        s.sink_chunks = (min(a.sinks, t.pmax + 1) + tb - 1) / tb;
        lo = max(0, t.pmin - a.window + 1);
    }
    s.first = max(lo / tb, s.sink_chunks);
    s.total = s.sink_chunks + max(0, t.pmax / tb - s.first + 1);
    return s;
}

__device__ __forceinline__ unsigned perm(unsigned hi, unsigned lo, unsigned sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ unsigned pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ void store4(float* p, f32x4 x) { *(f32x4*)p = x; }
__device__ __forceinline__ void store4(bf16* p, f32x4 x) { *(u32x2*)p = u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])}; }
__device__ __forceinline__ float lo_f(unsigned x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(unsigned x) { return __uint_as_float(x & 0xffff0000u); }

// global, not flat: a flat load would be waited for with every use of LDS
typedef const __attribute__((address_space(1))) unsigned mem_u32;
typedef const __attribute__((address_space(1))) u32x2 mem_u32x2;
typedef const __attribute__((address_space(1))) f32x4 mem_f32x4;
__device__ const u32x4 kv_zeros = {0, 0, 0, 0};                 // what dimensions past the head's size are read from, and rows that nobody sees

// ---- the cache types: how a wave holds one chunk of keys and values, and multiplies with it --------------------------------------------
// Scores are computed transposed, S^T = K Q^T with 16 keys x 16 columns per tile: lane (c, g) = (lane & 15, lane >> 4) reads key
// row c as the A operand, and gets in return the scores of column c with keys 4 g .. 4 g + 3.  Those are, register for register, the
// B operand of O^T = V^T P^T when the contraction takes the keys in that order, so probabilities never leave the lane; and because
// the order of the output rows is free too, lane (m, g) loads for the A operand the DV = DP / 16 consecutive dimensions m DV .. of its
// keys - whole rows, straight from memory - and transposes that small block in registers (one v_perm per two values).  Nothing
// passes through LDS.  A chunk is two tiles (32 keys) for bf16 and 4 bits, one (16 keys) for f32.  Where values are bf16 the products take
// probabilities in bf16 too, rounded once (their sum is of the unrounded ones): the rounding of each weight is averaged over the keys,
// the output's own is not (32 rows to 16 001 tokens: 1.8e-3 of the output against 1.7e-3 with fp32 weights).
template <typename T, int DP> struct Chunk;

template <int DP> struct Chunk<bf16, DP> {
    static constexpr int TILES = 2, NS = DP / 32, DV = DP / 16, VW = DV / 2;
    typedef bf16 act;
    struct Q { u32x4 f[NS]; };
    u32x4 k[2][NS];
    unsigned v[8][VW];
    static __device__ __forceinline__ void load_q(Q& q, const bf16* p, int D, int g, bool on) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            u32x2 x = {0, 0}, y = x;
            if (on && 32 * s + 8 * g < D) { x = *(const u32x2*)(p + 32 * s + 8 * g); y = *(const u32x2*)(p + 32 * s + 8 * g + 4); }
            q.f[s] = u32x4{x[0], x[1], y[0], y[1]};
        }
    }
    static __device__ __forceinline__ int row_bytes(int D) { return 2 * D; }
    static __device__ __forceinline__ int step_bytes() { return 0; }
    // tile: where row 0 of the 16 rows of tile u lies; dimensions past the head's size read its first ones (`scores` takes zeros for them)
    __device__ __forceinline__ void load_k(int u, const char* tile, const char*, int D, int g, int cq) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = 32 * s + 8 * g;
            k[u][s] = *(const u32x4*)(tile + (unsigned)(2 * (cq * D + (d < D ? d : 0))));
        }
    }
    __device__ __forceinline__ void load_v(int u, const char* tile, const char*, int D, int g, int m) {
        const unsigned off = (unsigned)(2 * (4 * g * D + (m * DV < D ? m * DV : 0)));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const char* p = tile + 2 * r * D;
            if constexpr (VW == 2) { const u32x2 x = *(const u32x2*)(p + off); v[4 * u + r][0] = x[0]; v[4 * u + r][1] = x[1]; }
            else
#pragma unroll
                for (int w = 0; w < VW; w += 4) {
                    const u32x4 x = *(const u32x4*)(p + off + 4 * w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * u + r][w + e] = x[e];
                }
        }
    }
    // keep(u, r): whether key 4 g + r of tile u counts.  An old NaN in a row that does not must not meet its probability 0.
    template <typename Keep> __device__ __forceinline__ void hide(int, Keep keep) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!keep(j >> 2, j & 3))
#pragma unroll
                for (int w = 0; w < VW; ++w) v[j][w] = 0;
    }
    // Past the head's size q is 0, but 0 times what a key has in another dimension is NaN where that is infinite.
    __device__ __forceinline__ f32x4 scores(int u, const Q& q, unsigned, int D, int g) const {
        f32x4 s = {0, 0, 0, 0};
        if (D == DP) {
#pragma unroll
            for (int i = 0; i < NS; ++i) s = mfma_bf16(k[u][i], q.f[i], s);
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) s = mfma_bf16(32 * i + 8 * g < D ? k[u][i] : u32x4{0, 0, 0, 0}, q.f[i], s);
        }
        return s;
    }
    __device__ __forceinline__ void weigh(const float* p, f32x4* o, unsigned) const {
        u32x4 b;
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = pack2(p[2 * j], p[2 * j + 1]);
#pragma unroll
        for (int i = 0; i < DV; ++i) {
            u32x4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = perm(v[2 * j + 1][i / 2], v[2 * j][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
            o[i] = mfma_bf16(x, b, o[i]);
        }
    }
    static __device__ __forceinline__ int dim(int i, int m) { return m * DV + i; }      // of row m of output tile i
    // a lane's values of one column: rows 4 g + r of all tiles
    template <typename E, typename Get> static __device__ __forceinline__ void store(E* out, int D, int g, Get get) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if ((4 * g + r) * DV < D)
#pragma unroll
                for (int i = 0; i < DV; i += 4) store4(out + (4 * g + r) * DV + i, f32x4{get(i, r), get(i + 1, r), get(i + 2, r), get(i + 3, r)});
    }
};

template <int DP> struct Chunk<float, DP> {
    static constexpr int TILES = 1, NS = DP / 16, DV = DP / 16;
    typedef float act;
    struct Q { f32x4 f[NS]; };
    f32x4 k[1][NS];
    f32x4 v[4][DV / 4];
    static __device__ __forceinline__ void load_q(Q& q, const float* p, int D, int g, bool on) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            q.f[s] = f32x4{0, 0, 0, 0};
            if (on && 16 * s < D) q.f[s] = *(const f32x4*)(p + 16 * s + 4 * g);
        }
    }
    static __device__ __forceinline__ int row_bytes(int D) { return 4 * D; }
    static __device__ __forceinline__ int step_bytes() { return 0; }
    __device__ __forceinline__ void load_k(int, const char* tile, const char*, int D, int g, int cq) {
        // past the head's size (D is a multiple of 16): zeros, as in bf16's scores, but from memory - a branch around the products there costs
        // the loads that run beside them (4 prompts of 2 048 tokens, 16 heads of 64: 425 us against 375)
#pragma unroll
        for (int s = 0; s < NS; ++s) k[0][s] = *(mem_f32x4*)((16 * s < D ? tile : (const char*)&kv_zeros) + (16 * s < D ? (unsigned)(4 * (cq * D + 4 * g + 16 * s)) : 0u));
    }
    __device__ __forceinline__ void load_v(int, const char* tile, const char*, int D, int g, int m) {
        const unsigned off = (unsigned)(4 * (4 * g * D + (m * DV < D ? m * DV : 0)));
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < DV / 4; ++w) v[r][w] = *(const f32x4*)(tile + 4 * r * D + off + 16 * w);
    }
    template <typename Keep> __device__ __forceinline__ void hide(int, Keep keep) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!keep(0, j))
#pragma unroll
                for (int w = 0; w < DV / 4; ++w) v[j][w] = f32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ f32x4 scores(int, const Q& q, unsigned, int, int) const {
        f32x4 s = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0][i][e], q.f[i][e], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void weigh(const float* p, f32x4* o, unsigned) const {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < DV; ++i) o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][i >> 2][i & 3], p[r], o[i], 0, 0, 0);
    }
    static __device__ __forceinline__ int dim(int i, int m) { return m * DV + i; }
    template <typename E, typename Get> static __device__ __forceinline__ void store(E* out, int D, int g, Get get) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if ((4 * g + r) * DV < D)
#pragma unroll
                for (int i = 0; i < DV; i += 4) store4(out + (4 * g + r) * DV + i, f32x4{get(i, r), get(i + 1, r), get(i + 2, r), get(i + 3, r)});
    }
};

// 4 bits: a half byte n + 8 under the exponent of 128 IS the bf16 number 128 + (n + 8) (7 fraction bits), one and-or per two values.
// Keys: the accumulator starts at -136 sum(q) of the group, so a group's product comes out as sum(q n) and is scaled by the key's step.
// Values: the step goes into the probability, p step in bf16, and a second product with the constant -136 takes the offset out
// again, chunk by chunk, from the same rounded numbers (one offset for a whole row would cancel against 136 times its sum).
struct Int4 {};
// v of lane `from` of this lane's row of 16 (a DPP operand of the instruction that takes it, not one of its own)
template <int from> __device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + from, 0xf, 0xf, true));
}
template <int N> struct Const { static constexpr int value = N; };
template <int I, int N, typename F> __device__ __forceinline__ void each(F f) {      // f(Const<I>()) .. f(Const<N - 1>())
    if constexpr (I < N) { f(Const<I>()); each<I + 1, N>(f); }
}
template <int D> struct Chunk<Int4, D> {
    static constexpr int TILES = 2, S = D / 32, DV = D / 16;        // S groups; a lane's keys: 4 S bytes, its values: S bytes a key
    static constexpr int SW = (4 * S + 15) / 16;                    // steps of a lane group's four keys, S each, one per lane of the row
    typedef bf16 act;
    struct Q { u32x4 f[S]; float bias[S]; };
    unsigned k[2][S], v[8][(S + 3) / 4];
    float ks[2][SW], vs[2][SW];
    static __device__ __forceinline__ void load_q(Q& q, const bf16* p, int, int g, bool on) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            u32x2 x = {0, 0}, y = x;
            if (on) { x = *(const u32x2*)(p + 32 * s + 4 * g); y = *(const u32x2*)(p + 32 * s + 16 + 4 * g); }
            q.f[s] = u32x4{x[0], x[1], y[0], y[1]};
            float t = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) t += lo_f(q.f[s][e]) + hi_f(q.f[s][e]);
            t += __shfl_xor(t, 16);
            t += __shfl_xor(t, 32);
            q.bias[s] = -136.f * t;
        }
    }
    template <int N> static __device__ __forceinline__ void load_dw(unsigned* d, const void* p) {
        if constexpr (N == 1) d[0] = *(const unsigned*)p;
        else if constexpr (N == 2) { const u32x2 x = *(const u32x2*)p; d[0] = x[0]; d[1] = x[1]; }
        else
#pragma unroll
            for (int w = 0; w < N; w += 4) {
                const u32x4 x = *(const u32x4*)((const char*)p + 4 * w);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[w + e] = x[e];
            }
    }
    static __device__ __forceinline__ int row_bytes(int) { return D / 2; }
    static __device__ __forceinline__ int step_bytes() { return 2 * S; }
    static __device__ __forceinline__ void load_steps(float* d, const char* p, int g, int cq) {
#pragma unroll
        for (int w = 0; w < SW; ++w) d[w] = (float)*(const bf16*)(p + (unsigned)(2 * (4 * g * S + (S == 2 ? cq & 7 : 16 * w + cq))));
    }
    __device__ __forceinline__ void load_k(int u, const char* tile, const char* steps, int, int g, int cq) {
        load_dw<S>(k[u], tile + (unsigned)(cq * (D / 2) + g * 4 * S));
        load_steps(ks[u], steps, g, cq);
    }
    __device__ __forceinline__ void load_v(int u, const char* tile, const char* steps, int, int g, int m) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const char* p = tile + (unsigned)(4 * g * (D / 2) + m * S) + r * (D / 2);
            if constexpr (S == 2) v[4 * u + r][0] = *(const unsigned short*)p;
            else load_dw<S / 4>(v[4 * u + r], p);
        }
        load_steps(vs[u], steps, g, m);
    }
    // keep(u, r): whether key 4 g + r of tile u counts.  Its step is what goes: a NaN there must not meet its probability 0.
    template <typename Keep> __device__ __forceinline__ void hide(int cq, Keep keep) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < SW; ++w)
                if (!keep(u, S == 2 ? (cq & 7) >> 1 : (16 * w + cq) / S)) vs[u][w] = 0.f;
    }
    __device__ __forceinline__ f32x4 scores(int u, const Q& q, unsigned magic, int, int) const {
        f32x4 t = {0, 0, 0, 0};
        each<0, S>([&](auto si) {
            constexpr int s = decltype(si)::value;
            u32x4 x;
#pragma unroll
            for (int e = 0; e < 2; ++e) {                           // bytes s of the lane's m = 4 g + 2 e and + 1
                unsigned z;
                if constexpr (S == 2) z = perm(0, k[u][e], 0x0c000c00u | (unsigned)(s + 2) << 16 | (unsigned)s);
                else z = perm(k[u][(2 * e + 1) * (S / 4) + s / 4], k[u][2 * e * (S / 4) + s / 4], 0x0c000c00u | (unsigned)(s % 4 + 4) << 16 | (unsigned)(s % 4));
                x[e] = (z & 0x000f000fu) | magic;
                x[e + 2] = ((z >> 4) & 0x000f000fu) | magic;
            }
            const f32x4 d = mfma_bf16(x, q.f[s], f32x4{q.bias[s], q.bias[s], q.bias[s], q.bias[s]});
            each<0, 4>([&](auto ri) {
                constexpr int r = decltype(ri)::value, i = r * S + s;
                t[r] = fmaf(row_lane<i % 16>(ks[u][i / 16]), d[r], t[r]);
            });
        });
        return t;
    }
    __device__ __forceinline__ void weigh(const float* p, f32x4* o, unsigned magic) const {
        const u32x4 off = {0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};       // -136
        each<0, S>([&](auto si) {
            constexpr int s = decltype(si)::value;
            u32x4 b, lo, hi;
            each<0, 4>([&](auto ji) {
                constexpr int j = decltype(ji)::value, u = j >> 1, i = 2 * (j & 1) * S + s, k = i + S;
                b[j] = pack2(row_lane<i % 16>(vs[u][i / 16]) * p[2 * j], row_lane<k % 16>(vs[u][k / 16]) * p[2 * j + 1]);
                const unsigned z = perm(v[2 * j + 1][s / 4], v[2 * j][s / 4], 0x0c000c00u | (unsigned)(s % 4 + 4) << 16 | (unsigned)(s % 4));
                lo[j] = (z & 0x000f000fu) | magic;
                hi[j] = ((z >> 4) & 0x000f000fu) | magic;
            });
            o[2 * s] = mfma_bf16(lo, b, mfma_bf16(off, b, o[2 * s]));
            o[2 * s + 1] = mfma_bf16(hi, b, mfma_bf16(off, b, o[2 * s + 1]));
        });
    }
    static __device__ __forceinline__ int dim(int i, int m) { return 16 * i + m; }
    template <typename E, typename Get> static __device__ __forceinline__ void store(E* out, int, int g, Get get) {
#pragma unroll
        for (int i = 0; i < DV; ++i) store4(out + 16 * i + 4 * g, f32x4{get(i, 0), get(i, 1), get(i, 2), get(i, 3)});
    }
};

// A matrix product spreads an infinite or NaN value row to columns that do not see it (0 times it is NaN).  So where a result is not finite and the
// tile's columns differ in what they see, columns are computed again with the rows that they do not see taken out: positions from .. to at a
// time, between which no such row enters or leaves.  Finite data never comes there, and a second look is taken only where it can change
// something: for columns whose weights are finite (if they are not, a score of the column's own is not, and every look gives NaN), and if
// one of the rows that only some columns see - from the second position to the last, and as many at the window's far end - is not finite.
// Whether the tile's position pmin + 1 + i sees the row that it is the first to see (i < pmax - pmin), or not the one that the position before
// is the last to see (i further on by that), and that row is not finite: where a run of positions ends.
template <typename T> __device__ __forceinline__ bool ends_run(const KvAttendArgs& a, const Tile& t, int hk, int W, int sinks, int i) {
    asm volatile("" : "+v"(i));                // what follows from it is made here, not carried through the kernel in registers
    const int differ = t.pmax - t.pmin, D = a.c.dim, tok = i < differ ? t.pmin + 1 + i : t.pmin - W + 1 + i - differ;
    if (i >= 2 * differ || tok < 0 || (i >= differ && tok < sinks)) return false;
    const int page = a.c.table[(long long)t.row * a.c.width + (tok >> a.c.ps_shift)];
    if ((unsigned)page >= (unsigned)a.c.pages) return false;
    const long long row = ((((long long)a.layer * a.c.pages + page) * a.c.heads + hk) << a.c.ps_shift) + (tok & ((1 << a.c.ps_shift) - 1));
    bool bad = false;
    if constexpr (__is_same(T, float)) {
        const u32x4* v = (const u32x4*)((const float*)a.c.v + row * D);
        for (int d = 0; d < D / 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= (v[d][e] & 0x7f800000u) == 0x7f800000u;
    } else {                                   // 4 bits: the steps
        const int words = __is_same(T, bf16) ? D / 2 : D / 64;
        const unsigned* v = __is_same(T, bf16) ? (const unsigned*)a.c.v + row * words : (const unsigned*)a.c.vs + row * words;
        for (int d = 0; d < words; ++d) bad |= (v[d] & 0x7f80u) == 0x7f80u || (v[d] & 0x7f800000u) == 0x7f800000u;
    }
    return bad;
}

// Work on one tile of columns and one kv head: chunks cb .. ce - 1 of those the tile sees, whole (`out`) or as a part of them (unnormalised
// sums, maxima and weights: `part`).
struct KvPart { float *sums, *ml; };           // [16][DP], [16][2]

// The workgroup's waves take the chunks in turn, each with a running maximum and sum of its own, and are joined through LDS at the end
// (WAVES = 4), or a wave has all of them and writes the result itself (WAVES = 1: no LDS, no barrier, waves on tiles of their own).  Bound
// by memory for single tokens: the next chunk's keys are requested before this one's softmax, its values before this one's scores.
template <typename T, int DP, bool P8, int WAVES, typename Part>
__device__ __forceinline__ void attend_part(const KvAttendArgs& a, const Tile& t, const Span& span, int hk, int cb, int ce, bool whole_row, Part part_of,
                                            float (*so)[16][DP + 4], float (*sm)[16], float (*sl)[16]) {
    typedef Chunk<T, DP> C;
    typedef typename C::act A;
    constexpr int TB = 16 * C::TILES, NT = DP / 16;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));              // made new for each part: what follows from it is not kept in registers from one to the next
    const int lane = tid & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cq = lane & 15, g = lane >> 4;
    const int G = a.group, D = a.c.dim, sh = a.c.ps_shift;
    const int col = t.col0 + cq, qtok = col / G;
    int mypos = col < t.ncols && t.row >= 0 ? t.first_pos + qtok : -1;
    if (mypos > t.pmax) mypos = -1;
    typename C::Q q;
    C::load_q(q, (const A*)a.q.p + (long long)(t.tok0 + qtok) * a.q.ts + (long long)(hk * G + col - qtok * G) * a.q.hs, D, g, mypos >= 0);

    // The table is read through the scalar cache (nothing in this launch writes it), apart from the vector loads and their order.  Pages of 16
    // tokens and more: the 16 rows of a tile lie in one page, so its address is the same for the wave and a lane adds a constant.  (P8: pages
    // of 8, two to a tile.)
    typedef const __attribute__((address_space(4))) int* Entries;
    const Entries table = (Entries)(unsigned long long)(a.c.table + (long long)max(t.row, 0) * a.c.width);
    const int in_page = (1 << sh) - 1, last_entry = a.c.width - 1, rb = C::row_bytes(D), sb = C::step_bytes();
    const unsigned page_rows = (unsigned)a.c.heads << sh;                      // rows of one page, all heads
    const long long head0 = ((long long)a.layer * a.c.pages * a.c.heads + hk) << sh;
    const char *kb = (const char*)a.c.k + head0 * rb, *vb = (const char*)a.c.v + head0 * rb;
    const char *ksb = (const char*)a.c.ks + head0 * sb, *vsb = (const char*)a.c.vs + head0 * sb;
    const int W = a.window > 0 ? min(a.window, 1 << 30) : 1 << 30, sinks = a.window > 0 ? a.sinks : 0;

    const float cs = a.scale_log2e;
    unsigned magic = 0x43004300u;              // two bf16 exponents of 128, kept in a register: an and-or takes one constant
    asm("" : "+v"(magic));
    int from = t.pmin, to = t.pmax;            // positions that are looked at: all, then runs of them for the columns of lanes `again`
    unsigned long long again = ~0ull;
    unsigned ends = 0;                         // bit i: a run ends behind position pmin + i
    for (;;) {
        const int vlo = from - W, vhi = to;    // a value row counts if vlo < its position <= vhi
        f32x4 o[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i] = f32x4{0, 0, 0, 0};
        float m = -INFINITY, l = 0.f;
        struct Pages { int lo[C::TILES], hi[C::TILES]; };                     // of a tile's rows 0 .. 7 and 8 .. 15
        auto entries = [&](int tb) {
            Pages e;
#pragma unroll
            for (int u = 0; u < C::TILES; ++u) {
                e.lo[u] = table[min((tb + 16 * u) >> sh, last_entry)];
                e.hi[u] = P8 ? table[min((tb + 16 * u + 8) >> sh, last_entry)] : e.lo[u];
            }
            return e;
        };
        auto good = [&](int e) { return (unsigned)e < (unsigned)a.c.pages; };
        auto row = [&](const char* base, int e, int first, int bytes) { return base + (unsigned long long)(good(e) ? (unsigned)e : 0u) * (page_rows * (unsigned)bytes) + first * bytes; };
        auto keys = [&](C& ch, const Pages& e, int tb) {
#pragma unroll
            for (int u = 0; u < C::TILES; ++u) {
                const int first = (tb + 16 * u) & in_page;
                if constexpr (!P8) {
                    ch.load_k(u, row(kb, e.lo[u], first, rb), row(ksb, e.lo[u], first, sb), D, g, cq);
                } else {
                    const int lo = e.lo[u], hi = e.hi[u], ek = cq & 8 ? hi : lo, ev = g & 2 ? hi : lo;
                    ch.load_k(u, row(kb, ek, -(cq & 8), rb), row(ksb, ev, -4 * (g & 2), sb), D, g, cq);
                }
            }
        };
        auto values = [&](C& ch, const Pages& e, int tb) {
#pragma unroll
            for (int u = 0; u < C::TILES; ++u) {
                const int first = (tb + 16 * u) & in_page;
                if constexpr (!P8) {
                    ch.load_v(u, row(vb, e.lo[u], first, rb), row(vsb, e.lo[u], first, sb), D, g, cq);
                } else {
                    const int lo = e.lo[u], hi = e.hi[u], ev = g & 2 ? hi : lo;
                    ch.load_v(u, row(vb, ev, -4 * (g & 2), rb), row(vsb, ev, -4 * (g & 2), sb), D, g, cq);
                }
            }
        };
        // one chunk, at token `now` with pages `e`: scores, `between`, softmax, values
        auto consume = [&](C& ch, const Pages& e, int now, auto between) {
            float x[4 * C::TILES];
#pragma unroll
            for (int u = 0; u < C::TILES; ++u) {
                const f32x4 s = ch.scores(u, q, magic, D, g);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[4 * u + r] = s[r];
            }
            between();
            bool whole = now + TB - 1 <= t.pmin && (now > t.pmax - W || now + TB - 1 < sinks);
#pragma unroll
            for (int u = 0; u < C::TILES; ++u) whole = whole && good(e.lo[u]) && good(e.hi[u]);
            if (!whole) {
                auto there = [&](int u) {
                    const int lo = e.lo[u], hi = e.hi[u];
                    return good(P8 && (g & 2) ? hi : lo);
                };
#pragma unroll
                for (int j = 0; j < 4 * C::TILES; ++j) {
                    const int tok = now + 16 * (j >> 2) + 4 * g + (j & 3);
                    const bool sees = there(j >> 2) && tok <= mypos && (tok > mypos - W || tok < sinks);
                    x[j] = sees ? x[j] : -INFINITY;
                }
                ch.hide(cq, [&](int u, int r) {
                    const int tok = now + 16 * u + 4 * g + r;
                    return there(u) && tok <= vhi && (tok > vlo || tok < sinks);
                });
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < 4 * C::TILES; ++j) top = fmaxf(top, x[j]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = fmaxf(m, top * cs), mu = mn == -INFINITY ? 0.f : mn;
            if (__any(mn > m)) {
                const float f = __builtin_amdgcn_exp2f(m - mu);
                l *= f;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[i] *= f;
            }
            m = mn;
#pragma unroll
            for (int j = 0; j < 4 * C::TILES; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], cs, -mu));
                l += x[j];
            }
            ch.weigh(x, o, magic);
        };
        int c = cb + wave;
        auto at = [&](int i) { return span.chunk(min(i, ce - 1)) * TB; };      // past the end: the last chunk again, and not looked at
        if (c < ce) {
            C ch;
            Pages p = entries(at(c));
            keys(ch, p, at(c));
            do {
                values(ch, p, at(c));
                const Pages next = entries(at(c + WAVES));
                consume(ch, p, at(c), [&] { keys(ch, next, at(c + WAVES)); });
                p = next;
            } while ((c += WAVES) < ce);
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (WAVES == 1) {
            if (col < t.ncols && (ends == 0 || (mypos >= from && mypos <= to))) {
                if (whole_row) {
                    const bool none = mypos < 0 || l == 0.f;
                    const float inv = 1.0f / l;
                    A* out = (A*)a.out + ((long long)(t.tok0 + qtok) * a.q_heads + hk * G + col - qtok * G) * D;
                    C::store(out, D, g, [&](int i, int r) { return none ? 0.f : o[i][r] * inv; });
                } else {
                    const KvPart part = part_of();
                    C::store(part.sums + cq * DP, D, g, [&](int i, int r) { return o[i][r]; });
                    if (g == 0) { part.ml[2 * cq] = mypos < 0 ? -INFINITY : m; part.ml[2 * cq + 1] = mypos < 0 ? 0.f : l; }
                }
            }
        } else if (ends == 0 || (mypos >= from && mypos <= to)) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) so[wave][cq][C::dim(i, 4 * g + r)] = o[i][r];
            if (g == 0) { sm[wave][cq] = mypos < 0 ? -INFINITY : m; sl[wave][cq] = mypos < 0 ? 0.f : l; }
        }
        if (ends == 0) {
            float bad = 0.f;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) bad += o[i][r] * 0.f;
            const int differ = t.pmax - t.pmin;                                     // below 16
            if (differ <= 0) break;
            again = __ballot(mypos >= 0 && bad != 0.f && l * 0.f == 0.f);
            if (!again) break;
            const unsigned long long rows = __ballot(ends_run<T>(a, t, hk, W, sinks, lane));
            ends = (unsigned)(rows | rows >> differ) & ((1u << differ) - 1);
            if (!ends) break;
            to = t.pmin - 1;
        }
        do {
            from = to + 1;
            const unsigned rest = from > t.pmax ? 0 : ends >> (from - t.pmin);
            to = rest ? from + __builtin_ctz(rest) : t.pmax;
        } while (from <= t.pmax && !(again & __ballot(mypos >= from && mypos <= to)));
        if (from > t.pmax) break;
    }
    if constexpr (WAVES == 1) return;
    __syncthreads();
    // join the four waves; thread (c, j) takes DP / 16 dimensions of column c
    const int c = tid >> 4, d0 = (tid & 15) * (DP / 16);
    if (t.col0 + c >= t.ncols || d0 >= D) return;
    float mx = -INFINITY, l = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm[w][c]);
    const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = __builtin_amdgcn_exp2f(sm[w][c] - mu);
        l = fmaf(sl[w][c], f[w], l);
    }
    f32x4 r[DP / 64];
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        r[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) r[i] += *(const f32x4*)&so[w][c][d0 + 4 * i] * f[w];
    }
    if (!whole_row) {
        const KvPart part = part_of();
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) *(f32x4*)(part.sums + c * DP + d0 + 4 * i) = r[i];
        if (d0 == 0) { part.ml[2 * c] = mx; part.ml[2 * c + 1] = l; }
        return;
    }
    const int tk = (t.col0 + c) / G, h = hk * G + t.col0 + c - tk * G;
    const bool none = l == 0.f;
    const float inv = 1.0f / l;
    A* out = (A*)a.out + ((long long)(t.tok0 + tk) * a.q_heads + h) * D + d0;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * i + e] = (A)(none ? 0.f : r[i][e] * inv);
}

// ---- single tokens: one new token per row, up to FLAT tiles --------------------------------------------------------------------------
// A launch of as many waves as run at once; all (tile, kv head, chunk) triples in one line, cut into that many equal runs.  So long rows and
// short ones, few and many, load the card alike, whatever the host does not know about lengths.  A wave's run touches whole (tile,
// head) pairs and at most two in part, its first and its last: two parts per wave are all the workspace there is, and
// kv_flat_join_kernel puts the parts together.  Each workgroup finds the line's layout by itself: the chunk counts of all tiles, summed up.
// A run for each wave rather than for each workgroup: no meeting of waves at a pair's end, which short rows have often (64 rows of 512
// tokens in 4 bits 24 us against 47, in bf16 31 against 44; 32 rows of 3200 - 16001 in bf16 226 us against 223: 5.5 TB/s; 64 such rows in 4 bits 164 us, 4.8 TB/s, where
// unpacking on the vector units is what is left).
constexpr int FLAT = 1024;
constexpr int FLAT_LEAST = 4;                  // chunks of a run

struct KvFlat {                                // the workspace (the entry point keeps the line below 2^31 chunks)
    int* before;                               // [tiles + 1] chunks of the tiles before, for one head
    float *sums, *ml;                          // parts [2 runs][min(16, group)][DP], [..][2]
    int cols;
    __host__ __device__ KvFlat(float* ws, int runs, int dp, int group) {
        before = (int*)ws;
        cols = group < 16 ? group : 16;
        sums = ws + FLAT + 4;
        ml = sums + 2ll * runs * cols * dp;
    }
    __host__ __device__ static size_t bytes(int runs, int dp, int group) {
        return (FLAT + 4 + 2ull * runs * (group < 16 ? group : 16) * (dp + 2)) * sizeof(float);
    }
};
__device__ __forceinline__ int kv_flat_run(int units, int runs) { return max((units + runs - 1) / runs, FLAT_LEAST); }
// a tile of single tokens, given its table row and length
__device__ __forceinline__ Tile kv_flat_tile(const KvAttendArgs& a, int x, int row, int len) {
    Tile t;
    const int per = (a.group + 15) / 16;
    t.on = true;
    t.seq = t.tok0 = per == 1 ? x : x / per;
    t.col0 = (x - t.seq * per) * 16;
    t.ncols = a.group;
    t.row = row >= 0 && row < a.c.rows ? row : -1;
    t.first_pos = len - 1;
    t.pmin = max(t.first_pos, 0);
    t.pmax = t.row < 0 ? -1 : min(t.first_pos, (a.c.width << a.c.ps_shift) - 1);
    return t;
}

// waves of a SIMD, by the registers the kernel needs
__host__ __device__ constexpr int flat_waves(bool four_bits, int dp) { return dp == 256 ? 1 : dp == 64 ? 4 : four_bits ? 3 : 2; }

template <typename T, int DP, bool P8>
__global__ void __launch_bounds__(256, flat_waves(__is_same(T, Int4), DP)) kv_flat_kernel(const KvAttendArgs a, int tiles) {
    typedef Chunk<T, DP> C;
    typedef typename C::act A;
    constexpr int TB = 16 * C::TILES;
    constexpr int PER = FLAT / 256;
    __shared__ int before[FLAT + 1], row_of[FLAT], len_of[FLAT], wave_sum[4], first_tile[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), runs = 4 * gridDim.x, heads = a.c.heads;
    const int per_token = (a.group + 15) / 16;
    int n[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {            // thread t counts the chunks of tiles PER t ..
        const int x = PER * tid + k;
        n[k] = 0;
        if (x < tiles) {
            const int row = a.b.rows[per_token == 1 ? x : x / per_token], len = row >= 0 && row < a.c.rows ? a.c.lens[row] : 0;
            row_of[x] = row;
            len_of[x] = len;
            n[k] = kv_span(a, kv_flat_tile(a, x, row, len), TB).total;
        }
        sum += n[k];
    }
    const int mine = sum;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(sum, k);
        if (lane >= k) sum += y;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sum += wave_sum[w];
    const int units = (wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3]) * heads, run = kv_flat_run(units, runs);
    int b = sum - mine;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int x = PER * tid + k;
        if (x <= tiles) {
            before[x] = b;
            if (blockIdx.x == 0) KvFlat(a.ws, runs, DP, a.group).before[x] = b;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int u = (4 * blockIdx.x + w) * run;
            if (b * heads <= u && u < (b + n[k]) * heads) first_tile[w] = x;
        }
        b += n[k];
    }
    if (tid == 255 && tiles == FLAT) {
        before[FLAT] = b;
        if (blockIdx.x == 0) KvFlat(a.ws, runs, DP, a.group).before[FLAT] = b;
    }
    __syncthreads();
    // tiles that see nothing at all lie nowhere on the line: their outputs are zeros
    for (int x = blockIdx.x; x < tiles; x += gridDim.x)
        if (before[x] == before[x + 1]) {
            const Tile t = kv_flat_tile(a, x, row_of[x], len_of[x]);
            const int cols = min(16, t.ncols - t.col0);
            for (int i = tid; i < heads * cols * a.c.dim; i += 256) {
                const int d = i % a.c.dim, c = i / a.c.dim % cols, hk = i / a.c.dim / cols;
                ((A*)a.out)[((long long)t.tok0 * a.q_heads + hk * a.group + t.col0 + c) * a.c.dim + d] = (A)0.f;
            }
        }
    const long long u = (long long)(4 * blockIdx.x + wave) * run;
    if (u >= units) return;
    int x = __builtin_amdgcn_readfirstlane(first_tile[wave]), left = min(run, units - (int)u), slot = 2 * (4 * blockIdx.x + wave);
    int len = __builtin_amdgcn_readfirstlane(before[x + 1] - before[x]);
    const int off = (int)u - __builtin_amdgcn_readfirstlane(before[x]) * heads;
    int hk = off / len, cb = off - hk * len;
    for (;;) {
        const int ce = min(len, cb + left);
        const Tile t = kv_flat_tile(a, x, __builtin_amdgcn_readfirstlane(row_of[x]), __builtin_amdgcn_readfirstlane(len_of[x]));
        attend_part<T, DP, P8, 1>(a, t, kv_span(a, t, TB), hk, cb, ce, cb == 0 && ce == len, [&]() {
            const KvFlat ws(a.ws, runs, DP, a.group);
            return KvPart{ws.sums + (long long)slot * ws.cols * DP, ws.ml + (long long)slot * ws.cols * 2};
        }, nullptr, nullptr, nullptr);
        left -= ce - cb;
        if (left <= 0) return;
        cb = 0;
        slot |= 1;
        if (++hk == heads) {
            hk = 0;
            do {
                ++x;
                len = __builtin_amdgcn_readfirstlane(before[x + 1] - before[x]);
            } while (len == 0);
        }
    }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the n parts of one tile and head, part s at place(s).  Sixteen lanes have a
// column: each looks at every sixteenth part's maximum, then sums its DP / 16 dimensions of all.
template <typename A, int DP, typename Place>
__device__ __forceinline__ void join_parts(const KvAttendArgs& a, const Tile& t, int hk, int n, const float* sums, const float* ml, int cols, Place place) {
    constexpr int N = DP / 16;
    const int tid = threadIdx.x, G = a.group, D = a.c.dim, c = tid >> 4, j = tid & 15, d0 = j * N;
    if (t.col0 + (c & ~3) >= t.ncols) return;                  // whole waves
    const int cc = min(c, cols - 1);
    float m = -INFINITY;
    for (int s = j; s < n; s += 16) m = fmaxf(m, ml[2 * (place(s) * cols + cc)]);
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
    const float mu = m == -INFINITY ? 0.f : m;
    float r[N], l = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const long long row = place(s) * cols + cc;
        const float f = __builtin_amdgcn_exp2f(ml[2 * row] - mu), ls = ml[2 * row + 1];
        l = fmaf(ls, f, l);
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const f32x4 x = *(const f32x4*)(sums + row * DP + d0 + e);
#pragma unroll
            for (int w = 0; w < 4; ++w) r[e + w] = fmaf(x[w], f, r[e + w]);
        }
    }
    if (t.col0 + c >= t.ncols || d0 >= D) return;
    const int tk = (t.col0 + c) / G, h = hk * G + t.col0 + c - tk * G;
    const bool none = l == 0.f;
    const float inv = 1.0f / l;
    A* out = (A*)a.out + ((long long)(t.tok0 + tk) * a.q_heads + h) * D + d0;
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = (A)(none ? 0.f : r[e] * inv);
}
template <typename A, int DP>
__global__ void __launch_bounds__(256) kv_flat_join_kernel(const KvAttendArgs a, int tiles, int runs) {
    const int x = blockIdx.x, hk = blockIdx.y;
    const KvFlat ws(a.ws, runs, DP, a.group);
    const int b0 = ws.before[x], len = ws.before[x + 1] - b0, run = kv_flat_run(ws.before[tiles] * a.c.heads, runs);
    if (len == 0) return;
    const int u = b0 * a.c.heads + hk * len, ra = u / run, rb = (u + len - 1) / run;
    if (ra == rb) return;
    const Tile t = kv_flat_tile(a, x, 0, 1);                    // columns only
    // the part of the run in which it begins is that run's first only if it begins with it
    const long long first = 2ll * ra + (u == ra * run ? 0 : 1);
    join_parts<A, DP>(a, t, hk, rb - ra + 1, ws.sums, ws.ml, ws.cols, [&](int s) { return s == 0 ? first : 2ll * (ra + s); });
}

// ---- few columns per request, or many requests --------------------------------------------------------------------------------------
// Bound by latency where it is called: 8 rows of 700 tokens in 4 bits 10.7 us (six rounds of four waves), one row under a window of 4096 7.9
// and 3.9 to join.  One workgroup = one tile of columns, one kv head, one share (`share` chunks) of those the tile sees; where a tile has more than one
// share kv_join_kernel joins them.  The workspace: for each (tile, kv head) the parts [splits], then how many there are.
struct KvShares {
    float *sums, *ml;
    int* used;
    __device__ __forceinline__ KvShares(const KvAttendArgs& a, int tiles, int dp, int tile, int hk) {
        const long long n = (long long)tiles * a.c.heads, i = (long long)tile * a.c.heads + hk, rows = (long long)a.splits * 16;
        sums = a.ws + i * rows * dp;
        ml = a.ws + n * rows * dp + i * rows * 2;
        used = (int*)(a.ws + n * rows * (dp + 2)) + i;
    }
};
template <typename T, int DP, bool P8>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) kv_attend_kernel(const KvAttendArgs a) {
    constexpr int TB = 16 * Chunk<T, DP>::TILES;
    __shared__ __attribute__((aligned(16))) float so[4][16][DP + 4];
    __shared__ float sm[4][16], sl[4][16];
    const Tile t = kv_tile(a, blockIdx.x, 16, threadIdx.x & 63);
    if (!t.on) return;
    const int hk = blockIdx.y, z = blockIdx.z;
    const Span span = kv_span(a, t, TB);
    if (z > 0 && z * a.share >= span.total) return;
    const bool shared = a.splits > 1 && span.total > a.share;
    if (a.splits > 1 && z == 0 && threadIdx.x == 0)
        *KvShares(a, gridDim.x, DP, blockIdx.x, hk).used = shared ? min(a.splits, (span.total + a.share - 1) / a.share) : 1;
    const int ce = shared && z + 1 < a.splits ? min(span.total, (z + 1) * a.share) : span.total;       // a bound on lengths that was too low: the last share's
    attend_part<T, DP, P8, 4>(a, t, span, hk, z * a.share, ce, !shared, [&]() {
        const KvShares ws(a, gridDim.x, DP, blockIdx.x, hk);
        return KvPart{ws.sums + z * 16ll * DP, ws.ml + z * 32ll};
    }, so, sm, sl);
}

// many pairs: a wave for each (tile, kv head), when `alone` below holds
template <typename T, int DP, bool P8>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) kv_short_kernel(const KvAttendArgs a) {
    const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = (int)(w / a.c.heads), hk = (int)(w - (long long)x * a.c.heads);
    const Tile t = kv_tile(a, x, 16, threadIdx.x & 63);
    if (!t.on) return;
    const Span span = kv_span(a, t, 16 * Chunk<T, DP>::TILES);
    attend_part<T, DP, P8, 1>(a, t, span, hk, 0, span.total, true, [] { return KvPart{nullptr, nullptr}; }, nullptr, nullptr, nullptr);
}
template <typename A, int DP>
__global__ void __launch_bounds__(256) kv_join_kernel(const KvAttendArgs a) {
    const KvShares ws(a, gridDim.x, DP, blockIdx.x, blockIdx.y);
    const Tile t = kv_tile(a, blockIdx.x, 16, threadIdx.x & 63);
    if (!t.on) return;
    const int used = *ws.used;
    if (used > 1) join_parts<A, DP>(a, t, blockIdx.y, used, ws.sums, ws.ml, 16, [](int s) { return (long long)s; });
}

// ---- prompts -----------------------------------------------------------------------------------------------------------------------------
// Many columns per request (prompts, long pieces; bf16 and 4 bits): bound by the matrix cores and the LDS that feeds them.  One
// workgroup = 128 columns of one request and kv head, 32 per wave; keys and values go through LDS in tiles of KT, two buffers
// deep: while a tile is multiplied the next one's rows are on their way (bf16: to LDS; 4 bits: to registers), and one barrier per tile hands them over.
// A wave computes S^T = K Q^T on 32 x 32 x 16 products, so that a lane holds scores of one column and its probabilities are, register
// for register, the B operand of O^T = V^T P^T; V^T comes from the row-major image by transposed LDS reads.  The probabilities' maximum
// is allowed to lag: the sums are rescaled only when a column's maximum has grown by more than 2^8 (fp32 sums and bf16 probabilities have
// the range), which a causal row does a few times in all.
// Workgroups of one (request, kv head) sit eight apart in launch order, heads fastest: on the eight XCDs, whose workgroups are dealt
// round robin, a head's keys stay in one L2.  Long columns start first.  16503 new tokens in 6 requests under a window of 2048 (bf16, 16 heads
// on 8 of 128): 250 us, 820 TFLOP/s of what is visible; the same on 16-column tiles 978.
// 4 bits: four bytes of the row = one 16-byte chunk; the order of dimensions in a row is then the packed one, which Q's load and the output's
// store follow.  Scores are sums of many terms, whose roundings would move a probability by several bf16 steps: keys n * step are
// fp16 operands, whose 11 bits hold the product of 3 and 8 bits exactly, each key divided by a power of two of its largest step that a
// score gets back in fp32, and each query by one of its own (errors below 2^-24 of the largest step and |q|: less than single tokens take
// with their -136).  Values are rounded to bf16: one more rounding of what a weighted mean averages, like that of its weights.
__device__ const u32x4 kv_eights = {0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u};      // 4 bits: n = 0
template <typename T, int DP> struct Row;                       // chunk ch of a row: 8 values as 16 bytes
template <int DP> struct Row<bf16, DP> {                       // goes to LDS as it is
    static constexpr float UP = 1.0f;
    struct Raw {};
    static __device__ __forceinline__ int dim(int d) { return d; }      // of place d of a row
};
template <int D> struct Row<Int4, D> {
    static constexpr int S = D / 32;
    static constexpr float UP = 16.0f;         // what values are divided by in LDS: a power of two
    struct Raw { unsigned x; u32x2 st; };
    static __device__ __forceinline__ const char* base(const void* p, long long row, int) { return (const char*)p + row * (D / 2); }
    static __device__ __forceinline__ const bf16* steps(const bf16* p, long long row) { return p + row * S; }
    // (`ch`'s steps of a row begin at 4 (ch & 1) where there are eight.)  No branch: a row that is not `ok` is read from constants that make zeros.
    static __device__ __forceinline__ void load(Raw& r, bool ok, const char* row, const bf16* steps, int ch) {
        const void *x = ok ? (const void*)(row + 4 * ch) : (const void*)&kv_eights, *st = ok ? (const void*)(steps + (S == 8 ? 4 * (ch & 1) : 0)) : (const void*)&kv_zeros;
        r.x = *(mem_u32*)x;
        if constexpr (S == 2) r.st[0] = *(mem_u32*)st;
        else r.st = *(mem_u32x2*)st;
    }
    // A key's power of two: 2^10 steps of the largest one's exponent (`biased`, 12 .. 253, so that it and its reciprocal are normal numbers)
    static __device__ __forceinline__ unsigned exponent(const Raw& r) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 top = __builtin_bit_cast(u16x2, r.st[0] & 0x7fff7fffu);
        if constexpr (S > 2) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, r.st[1] & 0x7fff7fffu));
        unsigned most = max((unsigned)top[0], (unsigned)top[1]);
        if constexpr (S == 8) most = max(most, (unsigned)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, true));    // the row's other steps
        return min(max(most >> 7, 12u), 253u);
    }
    static __device__ __forceinline__ float grown(unsigned biased) { return __uint_as_float((biased - 10) << 23); }      // what its scores are multiplied by
    // n * step / grown as fp16, exact (a step far below the largest one: to 2^-24)
    static __device__ __forceinline__ u32x4 key(const Raw& r, unsigned biased) {
        const unsigned lo = r.x & 0x0f0f0f0fu, hi = (r.x >> 4) & 0x0f0f0f0fu;
        const float f = __uint_as_float((264 - biased) << 23);
        u32x4 v;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const unsigned w = r.st[S == 2 ? 0 : b >> 1];
            const float st = (b & 1 ? hi_f(w) : lo_f(w)) * f, z = -8.0f * st;
            v[b] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(fmaf((float)(lo >> (8 * b) & 255u), st, z), fmaf((float)(hi >> (8 * b) & 255u), st, z)));
        }
        return v;
    }
    // n * step / UP as u * (step / UP) - 8 (step / UP) with u = n + 8, exact in one fma of a converted byte; UP keeps 8 steps from overflowing
    static __device__ __forceinline__ u32x4 value(const Raw& r) {
        const unsigned lo = r.x & 0x0f0f0f0fu, hi = (r.x >> 4) & 0x0f0f0f0fu;
        u32x4 v;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const unsigned w = r.st[S == 2 ? 0 : b >> 1];
            const float st = (b & 1 ? hi_f(w) : lo_f(w)) * (1.0f / UP), z = -8.0f * st;
            v[b] = pack2(fmaf((float)(lo >> (8 * b) & 255u), st, z), fmaf((float)(hi >> (8 * b) & 255u), st, z));
        }
        return v;
    }
    static __device__ __forceinline__ int dim(int d) {
        const int byte = d >> 1;
        return 32 * (byte % S) + 16 * (d & 1) + byte / S;
    }
};

template <int DP> __device__ __forceinline__ int lds_k(int row, int ch) { return 2 * DP * row + 16 * (ch ^ (DP == 64 ? (row >> 1) & 7 : row & 15)); }
template <int DP> __device__ __forceinline__ int lds_v(int row, int ch) { return 2 * DP * row + 16 * (ch ^ (DP == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2)); }

__device__ __forceinline__ float max_halves(float x) {           // over lanes l and l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes per lane from memory to LDS at `lds` (uniform) + 16 lane, outside the compiler's count of loads: `landed` waits for them.
// (M0 is a reserved register: the compiler gives it to no value, and takes it in no list of what an asm block changes.)
// (M0 belongs to no value of the compiler's; its own uses write it right before.)
__device__ __forceinline__ void to_lds(const char* base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void to_lds(const void* p, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(p), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void meet() {                        // a barrier that leaves loads in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ unsigned lds_of(const void* p) { return (unsigned)(unsigned long long)(lds_void*)p; }

// PAD: the head is smaller than DP.  Kernels of their own, so that the others have neither its branches nor its registers (one kernel for both: D = 80
// 118 us and D = 256 261 for 4 x 2 000 tokens, against 104 and 257).
template <typename T, int DP, int KT, bool PAD>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) kv_prompt_kernel(const KvAttendArgs a, int tiles) {
    typedef Row<T, DP> R;
    constexpr bool DMA = !__is_same(T, Int4);
    static_assert(DMA || !PAD, "4-bit heads have the sizes of the tiles");
    constexpr int RB = 2 * DP, NCH = DP / 8, KS = DP / 16, ND = DP / 32, NT = KT / 32, RP = 256 / NCH, NR = KT / RP, RW = RP / 4;
    __shared__ __attribute__((aligned(16))) unsigned char sk[2][KT * RB], sv[2][KT * RB];
    __shared__ unsigned long long again[4], ends[4];           // as in attend_part, in LDS: no register is left to carry them
    __shared__ __attribute__((aligned(16))) float grown[2][DMA ? 4 : KT];      // 4 bits: of each key of a tile
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.c.heads, G = a.group, D = PAD ? a.c.dim : DP, sh = a.c.ps_shift;
    const Tile t = kv_tile(a, tiles - 1 - (int)(blockIdx.x / a.c.heads), 128, lane);
    if (!t.on) return;
    const int r = lane & 31, hh = lane >> 5;
    const int col = t.col0 + 32 * wave + r, qtok = col / G;
    int mypos = col < t.ncols && t.row >= 0 ? t.first_pos + qtok : -1;
    if (mypos > t.pmax) mypos = -1;
    const int c0 = t.col0 + 32 * wave, c1 = min(c0 + 32, t.ncols) - 1;              // the wave's columns and the positions they span
    const int wmin = max(t.first_pos + c0 / G, 0), wmax = c1 < c0 || t.row < 0 ? -1 : min(t.first_pos + c1 / G, t.pmax);
    bf16x8 qf[KS];
    {
        const bf16* q = (const bf16*)a.q.p + (long long)(t.tok0 + qtok) * a.q.ts + (long long)(hk * G + col - qtok * G) * a.q.hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) qf[s][e] = (bf16)0.f;
            const int d = 16 * s + 8 * hh;
            if (mypos >= 0 && d < D) {
                if constexpr (!DMA) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) qf[s][e] = q[R::dim(d + e)];
                } else {
                    const bf16x4 x = *(const bf16x4*)(q + d), y = *(const bf16x4*)(q + d + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { qf[s][e] = x[e]; qf[s][4 + e] = y[e]; }
                }
            }
        }
    }
    float cs = a.scale_log2e;
    if constexpr (!DMA) {                      // this column's query as fp16, its largest dimension in 2^14 .. 2^15
        unsigned top = 0;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned w = __builtin_bit_cast(u32x4, qf[s])[e];
                top = max(top, max(w & 0x7fff0000u, w << 16 & 0x7fff0000u));
            }
        top = __float_as_uint(max_halves(__uint_as_float(top >> 1))) << 1;        // (shifted: no NaN among what a maximum of floats is taken of)
        const unsigned biased = max(top >> 23, 15u);
        const float f = __uint_as_float((268 - biased) << 23);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const u32x4 w = __builtin_bit_cast(u32x4, qf[s]);
            u32x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(lo_f(w[e]) * f, hi_f(w[e]) * f));
            qf[s] = __builtin_bit_cast(bf16x8, h);
        }
        // kept off 0 and infinity, which times a masked score or a score of 0 would be NaN
        cs = fminf(fmaxf(cs * __uint_as_float((biased - 14) << 23), 0x1p-126f), 0x1.fffffep127f);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));   // waited for here: a wait in the loop would be for every load in flight
    const Span span = kv_span(a, t, KT);
    const int* table = a.c.table + (long long)max(t.row, 0) * a.c.width;
    const long long page_rows = (long long)a.c.heads << sh, head0 = ((long long)a.layer * a.c.pages * a.c.heads + hk) << sh;
    const int in_page = (1 << sh) - 1, last_entry = a.c.width - 1, row_bytes = 2 * D;
    const unsigned page_bytes = (unsigned)page_rows * row_bytes;                   // below 2^32: the entry points see to it
    const char *kbase = (const char*)a.c.k + (DMA ? head0 * row_bytes : 0), *vbase = (const char*)a.c.v + (DMA ? head0 * row_bytes : 0);
    const int W = a.window > 0 ? min(a.window, 1 << 30) : 1 << 30, sinks = a.window > 0 ? a.sinks : 0;
    // This thread stages 16-byte slot `slot` of rows row0 + i RP; the rows of a wave and i are RW consecutive ones, which lie in one page.
    const int slot = tid & (NCH - 1), row0 = tid / NCH, sub = lane / NCH;
    // LDS places of this lane's operands; tiles, halves and buffers are constants added to them
    constexpr bool FEW = DP == 256;            // registers are short: places from the first one by exclusive or, where they are used
    int ak[FEW ? 1 : KS], av[FEW ? 1 : ND];
    {
        const int q4 = (lane >> 2) & 3, p4 = lane & 3, c16 = (lane >> 4) & 1;
#pragma unroll
        for (int k = 0; k < (FEW ? 1 : KS); ++k) ak[k] = lds_k<DP>(r, 2 * k + hh);
#pragma unroll
        for (int n = 0; n < (FEW ? 1 : ND); ++n) av[n] = lds_v<DP>(4 * hh + q4, 4 * n + 2 * c16 + (p4 >> 1)) + 8 * (p4 & 1);
    }

    auto key_at = [&](int k) { return FEW ? ak[0] ^ (32 * k) : ak[FEW ? 0 : k]; };
    auto value_at = [&](int n) { return FEW ? av[0] ^ (64 * n) : av[FEW ? 0 : n]; };

    // Past the head's size keys are zeros: q is 0 there, but 0 times an infinity would be NaN.  (Values: rows of the product that nobody stores.)
    if constexpr (PAD) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (lds_k<DP>(row0 + i * RP, slot) - RB * (row0 + i * RP) >= row_bytes)
#pragma unroll
                for (int b = 0; b < 2; ++b) *(u32x4*)(sk[b] + RB * (row0 + i * RP) + 16 * slot) = u32x4{0, 0, 0, 0};
    }
    int from = t.pmin, to = t.pmax;            // as in attend_part
    bool all = true;
    for (;;) {
        const int vlo = from - W, vhi = to;
        typename R::Raw kr[DMA ? 1 : NR], vr[DMA ? 1 : NR];
        // 64 entries of the table, one per lane, read again only when a tile leaves them: the wait for them is one for every load in flight
        int ent = 0, ent0 = -0x40000000;
        unsigned long long good = 0;           // which of them name a page of the pool
        long long place[DMA ? NR : 1];         // where this wave's rows of the tile last asked for begin, in bytes from a tensor's first
        int page[DMA ? 1 : NR];                // the pages of this thread's
        // Looks a tile's rows up; returns which of its keys have a page.
        auto find = [&](int c) -> unsigned long long {
            const int kb = span.chunk(c) * KT, e0 = kb >> sh;
            if (e0 < ent0 || ((kb + KT - 1) >> sh) > ent0 + 63) {
                ent0 = e0;
                ent = table[min(e0 + lane, last_entry)];
                asm volatile("" : "+v"(ent));                  // waited for here, not at every later use
                good = __ballot((unsigned)ent < (unsigned)a.c.pages);
            }
            if constexpr (DMA) {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int tok = kb + i * RP + wave * RW;
                    const unsigned p = (unsigned)__builtin_amdgcn_readlane(ent, (tok >> sh) - ent0);
                    place[i] = (long long)((unsigned long long)p * page_bytes) + (unsigned)((tok & in_page) * row_bytes);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NR; ++i) page[i] = __shfl(ent, ((kb + row0 + i * RP) >> sh) - ent0);
            }
            const int first = e0 - ent0, n = ((kb + KT - 1) >> sh) - e0 + 1;
            if ((~good >> first) & ((1ull << n) - 1)) return __ballot((good >> (((kb + (lane & (KT - 1))) >> sh) - ent0)) & 1);
            return ~0ull;
        };
        // Rows of one tensor of that tile on their way, to LDS (bf16) or to registers (4 bits: `stage` puts them there).  A row that no column
        // sees is read as zeros: its probabilities are 0, but 0 times an old NaN would still be NaN.
        auto fetch = [&](int c, unsigned long long okm, const char* base, const bf16* scales, unsigned char* lds, auto which, typename R::Raw* raw) {
            constexpr bool keys = decltype(which)::value;
            const int kb = span.chunk(c) * KT;
            if constexpr (DMA) {
                const bool inner = kb + KT - 1 <= vhi && (kb > vlo || kb + KT - 1 < sinks) && okm == ~0ull;
                // the chunk whose place this thread's slot is
                auto chunk = [&](int i) { return (keys ? lds_k<DP>(row0 + i * RP, slot) : lds_v<DP>(row0 + i * RP, slot)) - RB * (row0 + i * RP); };
                auto source = [&](int i) { return (unsigned)(sub * row_bytes + (!PAD || chunk(i) < row_bytes ? chunk(i) : 0)); };
                const unsigned to = lds_of(lds) + wave * RW * RB;
                if (inner && (!keys || !PAD)) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) to_lds(base + place[i], source(i), to + i * RP * RB);
                } else if (PAD && inner) {     // lanes past the head's size leave the zeros that lie there
#pragma unroll
                    for (int i = 0; i < NR; ++i)
                        if (chunk(i) < row_bytes) to_lds(base + place[i], source(i), to + i * RP * RB);
                } else {
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        const int first = i * RP + wave * RW, mine = kb + first + sub;
                        const bool ok = (okm >> first & 1) && mine <= vhi && (mine > vlo || mine < sinks) && (!keys || !PAD || chunk(i) < row_bytes);
                        to_lds(ok ? (const void*)(base + place[i] + source(i)) : (const void*)&kv_zeros, to + i * RP * RB);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int mine = kb + row0 + i * RP;
                    const bool ok = (unsigned)page[i] < (unsigned)a.c.pages && mine <= vhi && (mine > vlo || mine < sinks);
                    const long long at = head0 + (long long)page[i] * page_rows + (mine & in_page);
                    R::load(raw[i], ok, R::base(base, at, D), R::steps(scales, at), slot);
                }
            }
        };
        auto stage = [&](int buffer, bool keys, const typename R::Raw* raw) {
            if constexpr (!DMA) {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int row = row0 + i * RP;
                    if (keys) {
                        const unsigned biased = R::exponent(raw[i]);
                        *(u32x4*)(sk[buffer] + lds_k<DP>(row, slot)) = R::key(raw[i], biased);
                        if (slot == 0) grown[buffer][row] = R::grown(biased);
                    } else {
                        *(u32x4*)(sv[buffer] + lds_v<DP>(row, slot)) = R::value(raw[i]);
                    }
                }
            }
        };
        auto product = [&](bf16x8 x, bf16x8 q, f32x16 c) {
            if constexpr (DMA) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, q, c, 0, 0, 0);
            else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
        };
        // 4 bits: a tile's scores, multiplied by what its keys were divided by
        auto grow = [&](f32x16* s, const float* by) {
            if constexpr (!DMA) {
#pragma unroll
                for (int j = 0; j < 4 * NT; ++j) {
                    const f32x4 x = *(const f32x4*)(by + 8 * j + 4 * hh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j / 4][4 * (j % 4) + e] *= x[e];
                }
            }
        };
        f32x16 s[2][NT], o[ND];
        auto scores = [&](f32x16* s, const unsigned char* k0) {
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int u = 0; u < NT; ++u)
                    s[u] = product(*(const bf16x8*)(k0 + 32 * u * RB + key_at(k)), qf[k], s[u]);
        };
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
        float m = -INFINITY, l = 0.f;
        // A trip multiplies this tile's probabilities with its values while the next tile's scores are formed: the matrix cores have those to do
        // while the vector units do this tile's softmax.  So keys run one tile ahead of values, and both one tile behind their loads.
        unsigned long long ok0 = 0, ok1 = 0;   // keys of this tile and the next that have a page
        const Const<1> keys;
        const Const<0> values;
        if (span.total > 0) {
            ok0 = find(0);
            fetch(0, ok0, kbase, a.c.ks, sk[0], keys, kr);
            fetch(0, ok0, vbase, a.c.vs, sv[0], values, vr);
            stage(0, true, kr);
            stage(0, false, vr);
            if (span.total > 1) {
                ok1 = find(1);
                fetch(1, ok1, kbase, a.c.ks, sk[1], keys, kr);
                stage(1, true, kr);
            }
            landed();
            meet();
            scores(s[0], sk[0]);
            grow(s[0], grown[0]);
            meet();
        }
        auto tile = [&](int c, auto which) {
            constexpr int P = decltype(which)::value;
            const int kb = span.chunk(c) * KT;
            if constexpr (FEW) asm volatile("" : "+v"(ak[0]), "+v"(av[0]));
            const unsigned long long okm = ok0;
            if (c + 1 < span.total) fetch(c + 1, ok1, vbase, a.c.vs, sv[P ^ 1], values, vr);
            ok0 = ok1;
            if (c + 2 < span.total) {
                ok1 = find(c + 2);
                fetch(c + 2, ok1, kbase, a.c.ks, sk[P], keys, kr);
            }
            const bool whole = kb + KT - 1 <= wmin && (kb > wmax - W || kb + KT - 1 < sinks) && okm == ~0ull;
            if (!whole) {                      // key 32 u + 8 (i >> 2) + 4 hh + (i & 3), counted from kb + 32 u + 4 hh
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    const int from = kb + 32 * u + 4 * hh, hi = mypos - from, lo = mypos - W - from, sink = sinks - from;
                    const unsigned there = (unsigned)(okm >> (32 * u + 4 * hh));
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 8 * (i >> 2) + (i & 3);
                        s[P][u][i] = (there & 1u << key) && key <= hi && (key > lo || key < sink) ? s[P][u][i] : -INFINITY;
                    }
                }
            }
            float top = s[P][0][0];
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[P][u][i]);
            top = max_halves(top) * cs;
            if (__any(top > m + 8.0f)) {
                const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                l *= f;
#pragma unroll
                for (int n = 0; n < ND; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[n][i] *= f;
                m = mn;
            }
            const float mu = m == -INFINITY ? 0.f : m;
            // The order below is the order of the instructions: each matrix product has its operands' reads of LDS a few products earlier and a share of
            // the softmax's arithmetic behind it.  (Past the last tile the scores are of whatever lies there, and not looked at.)
            constexpr int QK = KS * NT, PV = 2 * NT * ND, NE = 16 * NT / 2, AHEAD = DMA ? 5 : 3;      // products, pairs of scores
            bf16x8 ring[AHEAD];
            u32x4 p[NT][2];
            auto read_k = [&](int j) { return *(const bf16x8*)(sk[P ^ 1] + 32 * (j % NT) * RB + key_at(j / NT)); };
            auto read_v = [&](int j) {
                bf16x8 x;
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    const unsigned char* ad = sv[P] + (16 * (j / ND) + 8 * jj) * RB + value_at(j % ND);
                    const bf16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)ad);
#pragma unroll
                    for (int w = 0; w < 4; ++w) x[4 * jj + w] = v[w];
                }
                return x;
            };
            auto weight = [&](int e) {         // scores 2 e, 2 e + 1 of this tile -> probabilities
                const int u = e >> 3, i = 2 * (e & 7);
                const float x = __builtin_amdgcn_exp2f(fmaf(s[P][u][i], cs, -mu)), y = __builtin_amdgcn_exp2f(fmaf(s[P][u][i + 1], cs, -mu));
                l += x + y;
                p[u][i >> 3][(i & 7) >> 1] = pack2(x, y);
            };
            auto read = [&](int j) { return j < QK ? read_k(j) : read_v(j - QK); };
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) ring[j] = read(j);
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[P ^ 1][u][i] = 0.f;
#pragma unroll
            for (int j = 0; j < QK + PV; ++j) {
                const bf16x8 x = ring[j % AHEAD];
                if (j < QK) s[P ^ 1][j % NT] = product(x, qf[j / NT], s[P ^ 1][j % NT]);
                else o[(j - QK) % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, __builtin_bit_cast(bf16x8, p[(j - QK) / ND / 2][((j - QK) / ND) & 1]), o[(j - QK) % ND], 0, 0, 0);
                if (j + AHEAD < QK + PV) ring[j % AHEAD] = read(j + AHEAD);
                if (j < QK)
#pragma unroll
                    for (int e = j * NE / QK; e < (j + 1) * NE / QK; ++e) weight(e);
                __builtin_amdgcn_sched_barrier(0);
            }
            grow(s[P ^ 1], grown[P ^ 1]);
            if (c + 2 < span.total) stage(P, true, kr);
            if (c + 1 < span.total) stage(P ^ 1, false, vr);
            landed();
            meet();
        };
        for (int c = 0; c < span.total; c += 2) {
            tile(c, Const<0>());
            if (c + 1 < span.total) tile(c + 1, Const<1>());
        }
        l += __shfl_xor(l, 32);
        if (col < t.ncols && (all || (mypos >= from && mypos <= to))) {
            const float inv = R::UP / l;
            const bool none = mypos < 0 || l == 0.f;
            bf16* out = (bf16*)a.out + ((long long)(t.tok0 + qtok) * a.q_heads + hk * G + col - qtok * G) * D;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * n + 8 * g + 4 * hh;
                    bf16x4 x;
#pragma unroll
                    for (int w = 0; w < 4; ++w) x[w] = (bf16)(none ? 0.f : o[n][4 * g + w] * inv);
                    if constexpr (!DMA) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) out[R::dim(d + w)] = x[w];
                    } else if (d < D) {
                        *(bf16x4*)(out + d) = x;
                    }
                }
        }
        if (all) {
            float bad = 0.f;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) bad += o[n][i] * 0.f;
            const int differ = t.pmax - t.pmin;                                     // below 128
            if (differ <= 0) return;
            const unsigned long long bits = __ballot(mypos >= 0 && bad != 0.f && l * 0.f == 0.f);
            if (lane == 0) again[wave] = bits;
            if (!__syncthreads_or(bits != 0)) return;
            const unsigned long long rows = __ballot(ends_run<T>(a, t, hk, W, sinks, tid));
            if (lane == 0) ends[wave] = rows;
            if (!__syncthreads_or(rows != 0)) return;
            all = false;
            to = t.pmin - 1;
        }
        do {
            from = to + 1;
            auto end = [&](int i) { return ends[i >> 6] >> (i & 63) & 1; };
            for (to = min(from, t.pmax); to < t.pmax && !end(to - t.pmin) && !end(to - t.pmin + t.pmax - t.pmin);) ++to;
            to = __builtin_amdgcn_readfirstlane(to);
        } while (from <= t.pmax && !__syncthreads_or((again[wave] & __ballot(mypos >= from && mypos <= to)) != 0));
        if (from > t.pmax) return;
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
long long tiles_of(int tokens, int sequences, int group, bool ragged, int cols = 16) {
    return ragged ? (long long)tokens * group / cols + sequences : (long long)sequences * ((group + cols - 1) / cols);
}
// Which kernel: 16-column tiles re-read a request's keys for every tile, but cut them over workgroups; 128-column ones feed them to four
// waves through LDS, and a row's keys stay with one workgroup.  The second kind needs enough columns per request to fill its tiles and
// enough (16-column tile, kv head) pairs that whole rows keep the card busy.  Measured, 128 columns against 16 (us; 16 heads on 8):
//   bf16, D = 128: 64 x 16 new tokens behind 984 (1024 pairs) 49 / 89, 2 x 1000 under a window of 500 (2000) 26 / 53, 6 x 64 behind 3936 (384)
//     90 / 121, 1 x 400 (400) 16 / 14, 1 x 100 (100) 10 / 6; of 16 columns: 300 x 8 behind 292 102 / 99, 700 x 8 behind 52 115 / 64
//   4 bits, where each workgroup has its own keys to unpack, D = 128: 24 x 500 (12000) 132 / 160, 64 x 128 behind 872 (8192) 215 / 233,
//     2 x 1000 under a window of 500 (2000) 43 / 38, 6 x 128 behind 3872 (768) 205 / 89, 1 x 400 (400) 31 / 12; of 128 columns a request:
//     64 x 64 (4096) 157 / 116
//   4 bits, D = 64: 24 x 500 (12000) 84 / 100; D = 256: 8 x 200 behind 3800 (1600) 389 / 514, 24 x 500 340 / 576, 3 x 235 (705) 42 / 30;
//     of 128 columns a request: 64 x 64 (4096) 464 / 386
bool prompts(const KvView& c, int tokens, int sequences, int q_heads, bool ragged) {
    if (c.dtype == Q3C_KV_F32 || !ragged) return false;
    const bool four = c.dtype == Q3C_KV_INT4;
    const long long columns = (long long)tokens * (q_heads / c.heads), least = !four ? 512 : c.dim == 256 ? 1536 : 6144;
    return columns >= (four ? 256ll : 32ll) * sequences && columns / 16 * c.heads >= least;
}
// The most chunks that a tile of `positions` neighbouring ones can see (of a row no longer than max_len, if that is given): its sinks', and those
// that window + positions - 1 tokens touch, which begin anywhere in a chunk.
long long most_chunks(const KvView& c, int window, int sinks, int max_len, int positions) {
    const int tb = c.dtype == Q3C_KV_F32 ? 16 : 32;
    long long len = (long long)c.width << c.ps_shift;
    if (max_len > 0 && max_len < len) len = max_len;
    long long n = len / tb + 1;
    if (window > 0) {
        const long long seen = ((long long)sinks + tb - 1) / tb + ((long long)window + positions - 1 + tb - 2) / tb + 1;
        if (seen < n) n = seen;
    }
    return n;
}
// Single tokens in a line of runs, unless the whole line is short: then the layout of the line costs more than it evens out (one row under a
// 4096-token window, 1040 chunks: 20 us against 14; 8 rows of 700 tokens in 4 bits: 17.6 against 11.5; 64 rows of 3200 - 16000: 184 against 218).
bool flat(const KvView& c, int sequences, int q_heads, bool ragged, int window, int sinks, int max_len) {
    const long long tiles = (long long)sequences * ((q_heads / c.heads + 15) / 16), line = tiles * c.heads * most_chunks(c, window, sinks, 0, 1);
    return !ragged && tiles <= FLAT && line < 0x70000000ll && tiles * c.heads * most_chunks(c, window, sinks, max_len, 1) > 8192;
}
// waves that run at once on 256 compute units
int flat_runs(const KvView& c) {
    return 1024 * flat_waves(c.dtype == Q3C_KV_INT4, padded_dim(c.dim));
}

}  // namespace

// How a tile's keys are cut otherwise: shares of as many chunks as make about 2048 workgroups of the longest rows there can be (eight per
// compute unit: short ones then even out what is left), of at least 8 chunks (two rounds of a workgroup's waves), no more than 256; rows of
// up to 32 chunks are left whole, since a second launch takes as long as six rounds (700 tokens: 11.5 us whole, 14.2 in shares of 8).
KvSplit q3_kv_attend_split(const KvView& c, int tokens, int sequences, int q_heads, bool ragged, int window, int sinks, int max_len) {
    if (flat(c, sequences, q_heads, ragged, window, sinks, max_len)) return KvSplit{0, 0, 0};
    if (prompts(c, tokens, sequences, q_heads, ragged)) return KvSplit{1, 0x7fffffff, 0};
    const int group = q_heads / c.heads;
    const long long chunks = most_chunks(c, window, sinks, max_len, ragged ? 16 : 1), base = tiles_of(tokens, sequences, group, ragged) * c.heads;
    long long share = (chunks * base + 2047) / 2048;
    if (share < 8) share = 8;
    if (share < (chunks + 255) / 256) share = (chunks + 255) / 256;
    share = (share + 3) / 4 * 4;
    KvSplit s;
    s.splits = base >= 2048 || chunks <= 32 ? 1 : (int)((chunks + share - 1) / share);
    s.share = s.splits == 1 ? 0x7fffffff : (int)share;
    s.most = (int)(chunks < 0x7fffffff ? chunks : 0x7fffffff);
    return s;
}
size_t q3_kv_attend_ws(const KvView& c, int tokens, int sequences, int q_heads, bool ragged, int splits) {
    const int group = q_heads / c.heads, dp = padded_dim(c.dim);
    if (splits == 0) return KvFlat::bytes(flat_runs(c), dp, group);
    if (splits == 1) return 0;
    return (size_t)(tiles_of(tokens, sequences, group, ragged) * c.heads) * ((size_t)splits * 16 * (dp + 2) + 1) * sizeof(float);
}

hipError_t q3_launch_kv_attend(const KvAttendArgs& a, hipStream_t s) {
    const unsigned tiles = (unsigned)tiles_of(a.b.tokens, a.b.sequences, a.group, a.b.offsets != nullptr);
    if (!tiles || !a.b.tokens) return hipSuccess;
    const dim3 grid(tiles, a.c.heads, a.splits ? a.splits : 1), join(tiles, a.c.heads);
    const int dp = padded_dim(a.c.dim), runs = a.splits ? 0 : flat_runs(a.c);
    if (prompts(a.c, a.b.tokens, a.b.sequences, a.q_heads, a.b.offsets != nullptr)) {
        const int n = (int)tiles_of(a.b.tokens, a.b.sequences, a.group, true, 128);
        const unsigned blocks = (unsigned)n * a.c.heads;
        if (a.c.dtype == Q3C_KV_BF16 && a.c.dim != dp) {
            if (dp == 64) kv_prompt_kernel<bf16, 64, 64, true><<<blocks, 256, 0, s>>>(a, n);
            else if (dp == 128) kv_prompt_kernel<bf16, 128, 64, true><<<blocks, 256, 0, s>>>(a, n);
            else kv_prompt_kernel<bf16, 256, 32, true><<<blocks, 256, 0, s>>>(a, n);
        } else if (a.c.dtype == Q3C_KV_BF16) {
            if (dp == 64) kv_prompt_kernel<bf16, 64, 64, false><<<blocks, 256, 0, s>>>(a, n);
            else if (dp == 128) kv_prompt_kernel<bf16, 128, 64, false><<<blocks, 256, 0, s>>>(a, n);
            else kv_prompt_kernel<bf16, 256, 32, false><<<blocks, 256, 0, s>>>(a, n);
        } else {
            if (dp == 64) kv_prompt_kernel<Int4, 64, 64, false><<<blocks, 256, 0, s>>>(a, n);
            else if (dp == 128) kv_prompt_kernel<Int4, 128, 32, false><<<blocks, 256, 0, s>>>(a, n);
            else kv_prompt_kernel<Int4, 256, 32, false><<<blocks, 256, 0, s>>>(a, n);
        }
        return hipGetLastError();
    }
    const long long pairs = (long long)tiles * a.c.heads;
    // A wave for each pair, with no meeting of waves, once there are pairs enough: for short rows (at most 16 chunks: four waves would have
    // four rounds) from one wave per SIMD on (1024 pairs: 128 tokens in bf16 7.5 us against 10.3 with four waves for each, 330 new tokens x 5
    // under a window of 72 in f32 15.7 against 21.6; 512 pairs of 64 tokens 6.5 against 6.0), for longer single tokens from eight (1100 rows
    // of 500 tokens in 4 bits 138 us against 175, bf16 410 against 409).  Not for longer pieces, whose tiles are as unlike as their
    // positions (4 x 2048 new tokens in f32: 433 us against 366).
    const bool alone = a.splits == 1 && ((a.most <= 16 && pairs >= 1024) || (!a.b.offsets && pairs >= 8192));
    const unsigned solo = alone ? (unsigned)((pairs + 3) / 4) : 0;
#define Q3_ATTEND(T, A, DP)                                                        \
    do {                                                                           \
        if (runs) {                                                                \
            if (a.c.ps_shift == 3) kv_flat_kernel<T, DP, true><<<runs / 4, 256, 0, s>>>(a, (int)tiles);  \
            else kv_flat_kernel<T, DP, false><<<runs / 4, 256, 0, s>>>(a, (int)tiles); \
            kv_flat_join_kernel<A, DP><<<join, 256, 0, s>>>(a, (int)tiles, runs);  \
        } else if (solo) {                                                         \
            if (a.c.ps_shift == 3) kv_short_kernel<T, DP, true><<<solo, 256, 0, s>>>(a);             \
            else kv_short_kernel<T, DP, false><<<solo, 256, 0, s>>>(a);            \
        } else {                                                                   \
            if (a.c.ps_shift == 3) kv_attend_kernel<T, DP, true><<<grid, 256, 0, s>>>(a);            \
            else kv_attend_kernel<T, DP, false><<<grid, 256, 0, s>>>(a);           \
            if (a.splits > 1) kv_join_kernel<A, DP><<<join, 256, 0, s>>>(a);       \
        }                                                                          \
    } while (0)
#define Q3_ATTEND_DIM(T, A)                        \
    do {                                           \
        if (dp == 64) Q3_ATTEND(T, A, 64);         \
        else if (dp == 128) Q3_ATTEND(T, A, 128);  \
        else Q3_ATTEND(T, A, 256);                 \
    } while (0)
    if (a.c.dtype == Q3C_KV_F32) Q3_ATTEND_DIM(float, float);
    else if (a.c.dtype == Q3C_KV_BF16) Q3_ATTEND_DIM(bf16, bf16);
    else Q3_ATTEND_DIM(Int4, bf16);
#undef Q3_ATTEND_DIM
#undef Q3_ATTEND
    return hipGetLastError();
}
