// Paged key/value cache of an autoregressive transformer: the per-head norm + rotation that fills it, reading it back, and the
// operations on its pages.  (The attention over it is kvattend.hip.)
//
// A page holds page_size tokens of every layer and head; a request's row of `table` lists its pages, `lens` its tokens, `refs[p]`
// how many table entries name page p (0: free).  Everything that a table, a row list or an offset says is checked where it is used:
// a bad entry costs the request its tokens and sets a bit of `status`, never an access outside the pool.
#include "kv.h"

namespace {

template <typename T, int N> using Vec = T __attribute__((ext_vector_type(N)));      // N elements as they lie in memory
template <int N> using Floats = float __attribute__((ext_vector_type(N)));

template <int N, typename T> __device__ __forceinline__ Vec<T, N> kv_load(const T* p) { return *(const Vec<T, N>*)p; }
template <int N, typename T> __device__ __forceinline__ void kv_store(T* p, Floats<N> v) { *(Vec<T, N>*)p = __builtin_convertvector(v, Vec<T, N>); }

// The value of the lane whose number differs in bit k (0 .. 3).  Bits 2 and 3 are taken by mirroring 8 or 16 lanes: right where the lanes
// that the lower bits tell apart hold one value, as in a butterfly that runs upwards.
template <typename V> __device__ __forceinline__ V lane_xor(V x, int k) {
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(V, k == 0   ? __builtin_amdgcn_update_dpp(0, i, 0xb1, 0xf, 0xf, true)
                                 : k == 1 ? __builtin_amdgcn_update_dpp(0, i, 0x4e, 0xf, 0xf, true)
                                 : k == 2 ? __builtin_amdgcn_update_dpp(0, i, 0x141, 0xf, 0xf, true)
                                          : __builtin_amdgcn_update_dpp(0, i, 0x140, 0xf, 0xf, true));
}
// the sum over each run of `lanes` (2 .. 32) lanes
__device__ __forceinline__ float sum_lanes(float x, int lanes) {
    x += lane_xor(x, 0);
    if (lanes > 2) x += lane_xor(x, 1);
    if (lanes > 4) x += lane_xor(x, 2);
    if (lanes > 8) x += lane_xor(x, 3);
    if (lanes > 16) x += __shfl_xor(x, 16);
    return x;
}

__device__ __forceinline__ void kv_flag(const KvView& c, int bits) { atomicOr(c.status, bits); }

// whether an earlier request of the call names the same table row: its tokens would race for the same places (wave-uniform)
__device__ __forceinline__ bool kv_repeated(const int* __restrict__ rows, int seq, int row, int lane) {
    for (int i = 0; i < seq; i += 64)
        if (__ballot(i + lane < seq && rows[min(i + lane, seq - 1)] == row)) return true;
    return false;
}
// the page of position pos, or -1
__device__ __forceinline__ int kv_page(const KvView& c, int row, int pos) {
    const int p = c.table[(long long)row * c.width + (pos >> c.ps_shift)];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}

// Where token `tok` goes: its position and page (-1: none).  false: nothing is to be done for it - it lies behind the last request, or has no
// valid row or position; then its queries are zeros.
__device__ __forceinline__ bool kv_place(const KvAppendArgs& a, int tok, bool first, int lane, int& pos, int& page, bool& zero) {
    int seq, row;
    zero = false;
    pos = kv_position(a.c, a.b, tok, lane, seq, row);
    if (first && lane == 0 && kv_ends_behind(a.b, tok)) kv_flag(a.c, Q3C_KV_BAD_ROW);
    if (pos < 0) {
        zero = pos != -1;
        if (zero && lane == 0 && first) kv_flag(a.c, Q3C_KV_BAD_ROW);
        return false;
    }
    page = kv_page(a.c, row, pos);
    if (page < 0 && lane == 0 && first) kv_flag(a.c, Q3C_KV_NO_PAGE);
    if (kv_repeated(a.b.rows, seq, row, lane)) {
        if (lane == 0 && first) kv_flag(a.c, Q3C_KV_BAD_ROW);
        page = -1;
    }
    return true;
}

// ---- append -----------------------------------------------------------------------------------------------------------------------
// y = x * rsqrt(mean(x^2) + eps) * w over a head's dimensions, then its first `rot` dimensions turned by the position's angle:
// (a, b) = (y_i, y_(i + rot/2)) -> (a cos - b sin, b cos + a sin); sums and products in fp32, one rounding at the store.  The keys
// and the (unchanged) values go straight to their page.  Bound by memory: 2 reads and writes of each element.
// A wave has one token and `parts`-th of its heads, VEC pairs per lane as two runs that are each other's rotation partners, so that the
// rotation needs no exchange between lanes and the norm one butterfly over the head's lanes.  Two runs of heads are requested before
// the token's place is looked up (offset -> row -> length -> page, four dependent reads): they are what a wave has to wait for once.
// 28144 tokens of 16 + 8 + 8 heads of 128 in bf16: 114 us, 4.2 TB/s; 64 single tokens 4.8 us.
template <typename T, int VEC, bool CACHED>     // CACHED: keys and values go to the pages here too (no 4-bit cache)
__device__ __forceinline__ void append_plain(const KvAppendArgs& a, int tok, int part, int parts, int lane, int lpu_shift) {
    constexpr int RUN = 2;
    const int D = a.c.dim, R = a.rot, H = a.q_heads, G = a.c.heads, units = CACHED ? H + 2 * G : H;
    const int lpu = 1 << lpu_shift, upw = 64 >> lpu_shift, ch = lane & (lpu - 1);
    const bool on = 2 * VEC * ch < D, in_turn = 2 * VEC * ch < R;
    int pos = 0, page = -1;
    for (int u0 = part * upw + (lane >> lpu_shift); u0 - (lane >> lpu_shift) < units; u0 += RUN * parts * upw) {
        Vec<T, VEC> x0[RUN], x1[RUN];
        int d0[RUN], d1[RUN], h[RUN], kind[RUN];
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int u = u0 + i * parts * upw;
            kind[i] = u >= units || !on ? 3 : u < H ? 0 : u < H + G ? 1 : 2;
            h[i] = u - (kind[i] == 0 ? 0 : kind[i] == 1 ? H : H + G);
            const bool turn = in_turn && kind[i] < 2;
            d0[i] = turn ? VEC * ch : 2 * VEC * ch;
            d1[i] = turn ? R / 2 + VEC * ch : 2 * VEC * ch + VEC;
            if (kind[i] < 3) {
                const KvStrided& src = kind[i] == 0 ? a.q : kind[i] == 1 ? a.k : a.v;
                const T* x = (const T*)src.p + tok * src.ts + h[i] * src.hs;
                x0[i] = kv_load<VEC>(x + d0[i]);
                x1[i] = kv_load<VEC>(x + d1[i]);
            } else {
                x0[i] = x1[i] = (T)0.f;
            }
        }
        if (u0 - (lane >> lpu_shift) == part * upw) {           // the first time round
            bool zero;
            if (!kv_place(a, tok, part == 0, lane, pos, page, zero)) {
                T* q = (T*)a.q_out + (long long)tok * H * D;
                if (zero)
                    for (int i = part * 64 + lane; i < H * D; i += parts * 64) q[i] = (T)0.f;
                return;
            }
        }
        Floats<VEC> co, si;
        if (in_turn) {
            co = *(const Floats<VEC>*)(a.cos_t + (long long)pos * (R / 2) + VEC * ch);
            si = *(const Floats<VEC>*)(a.sin_t + (long long)pos * (R / 2) + VEC * ch);
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            if (u0 - (lane >> lpu_shift) + i * parts * upw >= units) break;
            Floats<VEC> lo = __builtin_convertvector(x0[i], Floats<VEC>), hi = __builtin_convertvector(x1[i], Floats<VEC>);
            const float* w = kind[i] == 0 ? a.qw : kind[i] == 1 ? a.kw : nullptr;
            if (a.qw || a.kw) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
                ss = sum_lanes(ss, lpu);
                const float r = __builtin_amdgcn_rsqf(fmaf(ss, a.inv_dim, a.eps));
                if (w) {
                    lo = lo * r * *(const Floats<VEC>*)(w + d0[i]);
                    hi = hi * r * *(const Floats<VEC>*)(w + d1[i]);
                }
            }
            if (in_turn && kind[i] < 2) {
                const Floats<VEC> y0 = lo, y1 = hi;
                lo = y0 * co - y1 * si;
                hi = y1 * co + y0 * si;
            }
            T* y = nullptr;
            if (kind[i] == 0) y = (T*)a.q_out + ((long long)tok * H + h[i]) * D;
            else if (kind[i] < 3 && page >= 0)
                y = (T*)(kind[i] == 1 ? a.c.k : a.c.v) +
                    (((((long long)a.layer * a.c.pages + page) * G + h[i]) << a.c.ps_shift) + (pos & ((1 << a.c.ps_shift) - 1))) * D;
            if (y) { kv_store<VEC, T>(y + d0[i], lo); kv_store<VEC, T>(y + d1[i], hi); }
        }
    }
}

// x / d, rounded to nearest as the division is, with y = 1 / d rounded to nearest: the remainder of the first guess is exact in an fma, which
// makes the second one right (Markstein); d at least 2^-100 and the quotients below 2^20, so that nothing over- or underflows on the way.
__device__ __forceinline__ float divide(float x, float d, float y) {
    const float q = x * y;
    return fmaf(fmaf(-d, q, x), y, q);
}

// A 4-bit row: groups of 32 dimensions share step = bf16(absmax / 7); value n = rint(x / step) in -7 .. 7 is held as n + 8.  Byte
// [m][s] of the row (m < 16, s < dim / 32) packs dimensions 32 s + m (low half) and 32 s + 16 + m.  A lane has M neighbouring m of a
// head: whole bytes and, dim / 2 being a multiple of 16, both partners of its rotations.  The group maximum is taken on the bits of
// |x| (integers order like the floats, NaN above infinity), so a group that holds either reads back as NaN throughout.
// M = 4: 8-byte loads, two steps of each butterfly, 37 us for 10756 tokens of 16 + 8 + 8 heads of 128 (3.9 TB/s; 2: 39, 1: 45 us, where
// most of the time went to instructions).  A wave for a token's queries and one for its keys and values: both in one took 39 us.
constexpr int M4 = 4;                         // bytes of each group that a lane has: a head takes 16 / M4 lanes
template <int D>
__device__ __forceinline__ void append_int4(const KvAppendArgs& a, int tok, int unit0, int lane) {
    constexpr int N = D / 16, S = D / 32, M = M4, LPU = 16 / M;
    typedef Floats<M> F;
    const int G = a.c.heads, m = M * (lane % LPU), u = min(unit0 + lane / LPU, 2 * G - 1);
    const bool key = u < G, twin = unit0 + lane / LPU != u;          // twin: past the last head, a copy of it that stores nothing
    const int h = key ? u : u - G;
    const KvStrided& src = key ? a.k : a.v;
    const bf16* xp = (const bf16*)src.p + tok * src.ts + h * src.hs + m;
    Vec<bf16, M> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = kv_load<M>(xp + 16 * i);
    int pos, page;
    bool zero;
    if (!kv_place(a, tok, false, lane, pos, page, zero) || page < 0) return;
    F x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __builtin_convertvector(raw[i], F);
    if (key && a.kw) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j) ss = fmaf(x[i][j], x[i][j], ss);
        ss = sum_lanes(ss, LPU);
        const float r = __builtin_amdgcn_rsqf(fmaf(ss, a.inv_dim, a.eps));
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = x[i] * r * *(const F*)(a.kw + 16 * i + m);
    }
    if (key && a.rot) {
        const float* co = a.cos_t + (long long)pos * (D / 2) + m;
        const float* si = a.sin_t + (long long)pos * (D / 2) + m;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const F c = *(const F*)(co + 16 * i), s = *(const F*)(si + 16 * i), p = x[i], q = x[i + N / 2];
            x[i] = p * c - q * s;
            x[i + N / 2] = q * c + p * s;
        }
    }
    const long long at = ((((long long)a.layer * a.c.pages + page) * G + h) << a.c.ps_shift) + (pos & ((1 << a.c.ps_shift) - 1));
    Vec<unsigned, M * S / 4> bytes = 0;
    Vec<unsigned short, S> steps;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < M; ++j) top = max(top, max(__float_as_uint(x[2 * s][j]) & 0x7fffffffu, __float_as_uint(x[2 * s + 1][j]) & 0x7fffffffu));
#pragma unroll
        for (int k = 0; 1 << k < LPU; ++k) top = max(top, lane_xor<unsigned>(top, k));
        const bool plain = top - 0x0e000000u < 0x7f800000u - 0x0e000000u;      // 2^-99 .. finite
        const bf16 st = (bf16)(plain ? divide(__uint_as_float(top), 7.0f, 1.0f / 7.0f) : __uint_as_float(top) / 7.0f);
        const float step = (float)st, inv = 1.0f / step;
        steps[s] = __builtin_bit_cast(unsigned short, st);
        const bool some = step > 0.f && step < INFINITY;
#pragma unroll
        for (int j = 0; j < M; ++j) {
            const float x0 = x[2 * s][j], x1 = x[2 * s + 1][j];
            float n0, n1;
            if (step >= 0x1p-100f) {
                n0 = divide(x0, step, inv);
                n1 = divide(x1, step, inv);
            } else {
                n0 = x0 / step;
                n1 = x1 / step;
            }
            n0 = fminf(fmaxf(rintf(n0), -7.f), 7.f);
            n1 = fminf(fmaxf(rintf(n1), -7.f), 7.f);
            const unsigned byte = some ? (unsigned)((int)n0 + 8) | (unsigned)((int)n1 + 8) << 4 : 0x88u;
            bytes[(j * S + s) / 4] |= byte << (8 * ((j * S + s) & 3));
        }
    }
    if (twin) return;
    *(Vec<unsigned, M * S / 4>*)((unsigned char*)(key ? a.c.k : a.c.v) + at * (D / 2) + m * S) = bytes;
    if (m == 0) *(Vec<unsigned short, S>*)((unsigned short*)(key ? a.c.ks : a.c.vs) + at * S) = steps;
}

// `parts` waves have a token's heads (D4: its query heads; then one wave for each 4 * M4 of its key and value heads)
template <typename T, int VEC, int D4>      // D4: 0 = cache in T, else head size of a 4-bit cache
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs a, int parts, int waves, int lpu_shift) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = (int)(w / waves), part = (int)(w - (long long)tok * waves);
    if (tok >= a.b.tokens) return;
    if (D4 == 0 || part < parts) append_plain<T, VEC, D4 == 0>(a, tok, part, parts, lane, lpu_shift);
    else append_int4<D4 ? D4 : 64>(a, tok, (part - parts) * (4 * M4), lane);
}

// ---- gather: the stored keys and values of the same tokens, back in one piece (zeros where there is no page) -------------------------
// Bound by the wait for a token's place (four dependent reads) and by memory: a wave has up to RUN runs of a token's heads in flight (4 bits,
// 10756 tokens of 8 + 8 heads of 128 as bf16: 13.9 us against 16.3 with one run per wave; 4.1 TB/s).
template <typename T, typename O, int D4>
__global__ void __launch_bounds__(256) kv_gather_kernel(const KvView c, const KvBatch b, int layer, O* __restrict__ k_out, O* __restrict__ v_out,
                                                        int waves, int lpu_shift) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = (int)(w / waves), part = (int)(w - (long long)tok * waves);
    if (tok >= b.tokens) return;
    int seq, row;
    const int pos = kv_position(c, b, tok, lane, seq, row);
    if (part == 0 && lane == 0 && kv_ends_behind(b, tok)) kv_flag(c, Q3C_KV_BAD_ROW);
    if (pos == -1) return;
    const int page = pos < 0 ? -1 : kv_page(c, row, pos);
    if (pos < 0 && lane == 0 && part == 0) kv_flag(c, Q3C_KV_BAD_ROW);
    constexpr int S = D4 ? D4 / 32 : 2, RUN = D4 == 256 ? 2 : 4;
    const int lpu = 1 << lpu_shift, upw = 64 >> lpu_shift, ch = lane & (lpu - 1), s = ch >> 2, units = 2 * c.heads;
    const int in_page = pos & ((1 << c.ps_shift) - 1);
    for (int u0 = part * upw; u0 < units; u0 += RUN * waves * upw) {
        Vec<T, 8> x[RUN];
        Vec<unsigned, 4> w[RUN][S / 2];
        bf16 step[RUN];
#pragma unroll
        for (int r = 0; r < RUN; ++r) {
            const int u = u0 + r * waves * upw + (lane >> lpu_shift), h = u < c.heads ? u : u - c.heads;
            x[r] = (T)0.f;
            step[r] = (bf16)0.f;
#pragma unroll
            for (int i = 0; i < S / 2; ++i) w[r][i] = 0;
            if (u >= units || 8 * ch >= c.dim || page < 0) continue;
            const void* p = u < c.heads ? c.k : c.v;
            const long long at = ((((long long)layer * c.pages + page) * c.heads + h) << c.ps_shift) + in_page;
            if (D4 == 0) {
                x[r] = kv_load<8>((const T*)p + at * c.dim + 8 * ch);
            } else {                                           // dimensions 8 ch .. + 7: one half of byte s of eight neighbouring m's S bytes
#pragma unroll
                for (int i = 0; i < S / 2; ++i) w[r][i] = *(const Vec<unsigned, 4>*)((const unsigned char*)p + at * (16 * S) + (ch & 1) * 8 * S + 16 * i);
                step[r] = (u < c.heads ? c.ks : c.vs)[at * S + s];
            }
        }
#pragma unroll
        for (int r = 0; r < RUN; ++r) {
            const int u = u0 + r * waves * upw + (lane >> lpu_shift), h = u < c.heads ? u : u - c.heads;
            if (u >= units || 8 * ch >= c.dim) continue;
            Floats<8> y = __builtin_convertvector(x[r], Floats<8>);
            if (D4) {
                const int shift = 8 * (s & 3) + ((ch & 2) ? 4 : 0);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned v = S == 2   ? w[r][0][i >> 1] >> (16 * (i & 1))
                                       : S == 4 ? w[r][i >> 2 & (S / 2 - 1)][i & 3]
                                       : s < 4  ? w[r][i >> 1 & (S / 2 - 1)][2 * i & 3]
                                                : w[r][i >> 1 & (S / 2 - 1)][(2 * i + 1) & 3];
                    y[i] = page < 0 ? 0.f : (float)((int)(v >> shift & 15u) - 8) * (float)step[r];
                }
            }
            kv_store<8, O>((u < c.heads ? k_out : v_out) + ((long long)tok * c.heads + h) * c.dim + 8 * ch, y);
        }
    }
}

// ---- pages ----------------------------------------------------------------------------------------------------------------------------
// One workgroup plans each operation, so that page numbers come out the same whatever runs beside it: free pages are handed out
// lowest first, to requests in the order of the call.  That bounds its time by a few dependent reads of memory, not by bandwidth:
// 6.3 us for a token of each of 64 rows, 12.5 for 120 forks, 8.2 for a compaction of 1 900 pages.
constexpr int PLAN_T = 1024, PLAN_K = 8;      // a scan step looks at PLAN_T * PLAN_K pages

// Exclusive prefix sums of one value per thread over the workgroup, and its total.  `sums`: 17 ints of LDS.
__device__ __forceinline__ int plan_scan(int v, int* sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(x, k);
        if (lane >= k) x += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < PLAN_T / 64; ++i) {
        const int s = sums[i];
        if (i < wave) before += s;
        total += s;
    }
    return before + x - v;
}

// Calls take(rank, page) once for each of the pages in [from, to) that pred(page's count) holds for, ranks ascending with the page from
// `rank0`, until `most` have been taken; returns how many there were up to there (block-uniform).  PLAN_K counts per thread are
// read at once, in page order by (k, thread): a ballot ranks a wave's pages, a scan of the 128 ballots' counts the rest.
template <typename Pred, typename Take>
__device__ __forceinline__ int plan_pages(const KvView& c, int from, int to, int most, int* lds /* 17 + PLAN_K * 16 */, Pred pred, Take take) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* cnt = lds + 17;
    int done = 0;
    for (long long p0 = from; p0 < to && done < most; p0 += PLAN_T * PLAN_K) {
        unsigned long long bal[PLAN_K];
        int r[PLAN_K];
#pragma unroll
        for (int k = 0; k < PLAN_K; ++k) r[k] = c.refs[min(p0 + k * PLAN_T + tid, (long long)to - 1)];
#pragma unroll
        for (int k = 0; k < PLAN_K; ++k) bal[k] = __ballot(p0 + k * PLAN_T + tid < to && pred(r[k]));
        __syncthreads();
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < PLAN_K; ++k) cnt[k * 16 + wave] = __popcll(bal[k]);
        __syncthreads();
        int total;
        const int ex = plan_scan(tid < PLAN_K * 16 ? cnt[tid] : 0, lds, total);
        __syncthreads();
        if (tid < PLAN_K * 16) cnt[tid] = ex;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PLAN_K; ++k)
            if (bal[k] >> lane & 1) {
                const int rank = done + cnt[k * 16 + wave] + __popcll(bal[k] & ((1ull << lane) - 1));
                if (rank < most) take(rank, (int)(p0 + k * PLAN_T + tid));
            }
        done += total;
    }
    __syncthreads();
    return min(done, most);
}

// largest i with base[i] <= rank, base ascending, base[0] = 0 (entries of equal base: the last)
__device__ __forceinline__ int plan_owner(const int* base, int n, int rank) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (base[mid] <= rank) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Walk of threads 0 .. live - 1 over a list in LDS tiles (the whole workgroup calls it): each(j, list[j]) for all j < count.  Waves that have
// none of those threads only help to load: the comparisons of all sixteen would take most of a plan's time (120 pairs: 15 us against 13).
template <typename Each>
__device__ __forceinline__ void plan_walk(const int* __restrict__ list, int count, int live, int* tile /* PLAN_T, 16-byte aligned */, Each each) {
    for (int j0 = 0; j0 < count; j0 += PLAN_T) {
        const int n = min(PLAN_T, count - j0);
        __syncthreads();
        if ((int)threadIdx.x < n) tile[threadIdx.x] = list[j0 + threadIdx.x];
        __syncthreads();
        if ((int)(threadIdx.x & ~63u) >= live) continue;
        for (int j = 0; j < n; j += 4) {
            const int4 v = *(const int4*)(tile + j);
            each(j0 + j, v.x);
            if (j + 1 < n) each(j0 + j + 1, v.y);
            if (j + 2 < n) each(j0 + j + 2, v.z);
            if (j + 3 < n) each(j0 + j + 3, v.w);
        }
    }
    __syncthreads();
}

__global__ void __launch_bounds__(PLAN_T) kv_reserve_kernel(const KvView c, const KvBatch b) {
    __shared__ int lds[17 + PLAN_K * 16], base[PLAN_T], first[PLAN_T], row_of[PLAN_T];
    __shared__ __attribute__((aligned(16))) int tile[PLAN_T];
    const int tid = threadIdx.x;
    for (int s0 = 0; s0 < b.sequences; s0 += PLAN_T) {
        const int n = min(PLAN_T, b.sequences - s0), i = s0 + tid;
        int need = 0, row = tid < n ? b.rows[i] : -1, old = 0, add = 1;
        bool ok = row >= 0 && row < c.rows;
        if (ok) old = max(c.lens[row], 0);
        if (tid < n && b.offsets) {
            const int end = b.offsets[i + 1];
            add = min(max(end, 0), b.tokens) - min(max(b.offsets[i], 0), b.tokens);
            if (end > b.tokens) kv_flag(c, Q3C_KV_BAD_ROW);
        }
        plan_walk(b.rows, s0 + n, n, tile, [&](int j, int r) { ok = ok && (j >= i || r != row); });   // named twice: the first counts
        if (tid < n) {
            ok = ok && add >= 0;
            if (ok) {
                // a length may pass the row's table: those tokens have no place, append drops them and nobody sees them
                const long long cap = (long long)c.width << c.ps_shift, len = min((long long)old + add, 0x7fffffffll);
                if (len > cap) kv_flag(c, Q3C_KV_FULL_ROW);
                const int pm = (1 << c.ps_shift) - 1;
                first[tid] = (int)((min((long long)old, cap) + pm) >> c.ps_shift);
                need = (int)((min(len, cap) + pm) >> c.ps_shift) - first[tid];
                c.lens[row] = (int)len;
            } else {
                kv_flag(c, Q3C_KV_BAD_ROW);
            }
            row_of[tid] = row;
        }
        int total;
        const int ex = plan_scan(tid < n ? need : 0, lds, total);
        if (tid < n) base[tid] = ex;
        __syncthreads();
        const int got = plan_pages(c, 0, c.pages, total, lds, [](int r) { return r == 0; }, [&](int rank, int p) {
            const int o = plan_owner(base, n, rank);
            c.refs[p] = 1;
            c.table[(long long)row_of[o] * c.width + first[o] + rank - base[o]] = p;
        });
        // what the pool could not give stays without a page: such tokens are dropped by append and seen by nobody
        for (int r = got + tid; r < total; r += PLAN_T) {
            const int o = plan_owner(base, n, r);
            c.table[(long long)row_of[o] * c.width + first[o] + r - base[o]] = -1;
        }
        if (got < total && tid == 0) kv_flag(c, Q3C_KV_NO_PAGE);
        __syncthreads();
    }
}

// Gives pages back: a whole row's (its length becomes 0), or (trim) those that no further query of a sliding window sees - every
// token behind the first `sinks` and at least `window` before the row's end.  The exchange makes each table entry count once, whatever
// rows the call names twice; integer counts come out the same in any order.
__global__ void __launch_bounds__(256) kv_release_kernel(const KvView c, const int* __restrict__ rows, int trim, int window, int sinks) {
    const int row = rows[blockIdx.x];
    if (row < 0 || row >= c.rows) {
        if (threadIdx.x == 0 && blockIdx.y == 0) kv_flag(c, Q3C_KV_BAD_ROW);
        return;
    }
    if (!trim && blockIdx.y == 0 && threadIdx.x == 0) c.lens[row] = 0;
    const long long left = trim ? (long long)c.lens[row] - window : 0;      // trim: pages end by here
    for (int j = blockIdx.y * 256 + threadIdx.x; j < c.width; j += gridDim.y * 256) {
        if (trim) {
            const long long begin = (long long)j << c.ps_shift, end = begin + (1 << c.ps_shift);
            if (begin < sinks || end > left) continue;
        }
        int* e = c.table + (long long)row * c.width + j;
        if (*e < 0) continue;
        const int p = atomicExch(e, -1);
        if (p < 0) continue;
        if (p >= c.pages) kv_flag(c, Q3C_KV_BAD_PAGE);
        else if (atomicSub(c.refs + p, 1) <= 0) { atomicAdd(c.refs + p, 1); kv_flag(c, Q3C_KV_BAD_PAGE); }
    }
}

// fork, first launch: which pairs are good, and a free page for each partly filled last one.  ws: [count] source page or -1, [count]
// destination page, [count] 1 = good pair.
__global__ void __launch_bounds__(PLAN_T) kv_fork_plan_kernel(const KvView c, const int* __restrict__ parents, const int* __restrict__ children,
                                                              int count, int* __restrict__ ws) {
    __shared__ int lds[17 + PLAN_K * 16], taker[PLAN_T];             // taker: of the page of each rank
    __shared__ __attribute__((aligned(16))) int tile[PLAN_T];
    const int tid = threadIdx.x;
    for (int s0 = 0; s0 < count; s0 += PLAN_T) {
        const int n = min(PLAN_T, count - s0), i = s0 + tid;
        int need = 0;
        const int up = tid < n ? parents[i] : -1, ch = tid < n ? children[i] : -1;
        bool ok = up >= 0 && up < c.rows && ch >= 0 && ch < c.rows;
        if (ok) ok = c.lens[ch] == 0;
        // a child must be empty and named once (the first counts), and no row of the call both parent and child
        plan_walk(children, count, n, tile, [&](int j, int r) { ok = ok && (j >= i || r != ch) && r != up; });
        if (tid < n) {
            int src = -1;
            if (ok) {
                const int len = min(max(c.lens[up], 0), c.width << c.ps_shift);
                if (len & ((1 << c.ps_shift) - 1)) src = kv_page(c, up, len - 1);
            } else {
                kv_flag(c, Q3C_KV_BAD_ROW);
            }
            need = src >= 0;
            ws[i] = src;
            ws[count + i] = -1;
            ws[2 * count + i] = ok;
        }
        int total;
        const int ex = plan_scan(need, lds, total);
        if (need) taker[ex] = tid;
        __syncthreads();
        const int got = plan_pages(c, 0, c.pages, total, lds, [](int r) { return r == 0; }, [&](int rank, int p) {
            c.refs[p] = 1;
            ws[count + s0 + taker[rank]] = p;
        });
        if (tid < n && need && ex >= got) ws[i] = -1;
        if (got < total && tid == 0) kv_flag(c, Q3C_KV_NO_PAGE);
        __syncthreads();
    }
}

// ---- moving pages -----------------------------------------------------------------------------------------------------------------------
// A pair's work is cut into pieces of at most 16 KB of one (layer, tensor): 256 lanes x 16 bytes x 4 in flight.  685 MB of moved pages: 285 us,
// 4.8 TB/s read and written, what a large copy reaches.
struct KvPieces { int per_page[4]; long long bytes[4]; char* base[4]; int per_layer, layers, pages; };

__host__ __device__ __forceinline__ KvPieces kv_pieces(const KvView& c) {
    const long long tok = (long long)c.heads << c.ps_shift;
    const long long kv = c.dtype == Q3C_KV_INT4 ? tok * c.dim / 2 : tok * c.dim * (c.dtype == Q3C_KV_BF16 ? 2 : 4);
    const long long st = c.dtype == Q3C_KV_INT4 ? tok * (c.dim / 32) * 2 : 0;
    KvPieces p;
    p.bytes[0] = p.bytes[1] = kv;
    p.bytes[2] = p.bytes[3] = st;
    p.base[0] = (char*)c.k; p.base[1] = (char*)c.v; p.base[2] = (char*)c.ks; p.base[3] = (char*)c.vs;
    p.per_layer = 0;
    for (int t = 0; t < 4; ++t) { p.per_page[t] = (int)((p.bytes[t] + 16383) >> 14); p.per_layer += p.per_page[t]; }
    p.layers = c.layers;
    p.pages = c.pages;
    return p;
}
__device__ __forceinline__ void kv_copy_piece(const KvPieces& p, int piece, int src, int dst) {
    const int layer = piece / p.per_layer;
    int r = piece - layer * p.per_layer, t = 0;
    while (r >= p.per_page[t]) r -= p.per_page[t++];
    const long long n = p.bytes[t], off = (long long)r << 14;
    const uint4* s = (const uint4*)(p.base[t] + ((long long)layer * p.pages + src) * n + off);
    uint4* d = (uint4*)(p.base[t] + ((long long)layer * p.pages + dst) * n + off);
    const int q = (int)(min(n - off, 16384ll) >> 4), tid = threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (k * 256 + tid < q) v[k] = s[k * 256 + tid];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (k * 256 + tid < q) d[k * 256 + tid] = v[k];
}

// fork, second launch: a pair's first block writes the child's table row and counts, its others copy the page
__global__ void __launch_bounds__(256) kv_fork_kernel(const KvView c, const KvPieces pc, const int* __restrict__ parents,
                                                      const int* __restrict__ children, int count, const int* __restrict__ ws) {
    const int per = 1 + pc.layers * pc.per_layer, i = blockIdx.x / per, part = blockIdx.x - i * per;
    if (!ws[2 * count + i]) return;
    const int src = ws[i], dst = ws[count + i];
    if (part > 0) {
        if (src >= 0) kv_copy_piece(pc, part - 1, src, dst);
        return;
    }
    const int len = min(max(c.lens[parents[i]], 0), c.width << c.ps_shift), full = len >> c.ps_shift;
    const int* from = c.table + (long long)parents[i] * c.width;
    int* to = c.table + (long long)children[i] * c.width;
    for (int j = threadIdx.x; j < c.width; j += 256) {
        int p = j < full ? from[j] : j == full ? dst : -1;
        if (j < full && p >= 0) {
            if (p < c.pages) atomicAdd(c.refs + p, 1);
            else { kv_flag(c, Q3C_KV_BAD_PAGE); p = -1; }
        }
        to[j] = p;
    }
    if (threadIdx.x == 0) c.lens[children[i]] = len;
}

// Which pairs of a copy are done: the last of those that name one destination; none whose page is outside the pool, and none whose
// source is another pair's destination (the order of their copies would show).  ws[i] = source or -1.
__global__ void __launch_bounds__(256) kv_pairs_kernel(const KvView c, const int* __restrict__ src, const int* __restrict__ dst, int count,
                                                       int* __restrict__ ws) {
    __shared__ int tile[256];
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int s = i < count ? src[i] : -1, d = i < count ? dst[i] : -1;
    bool ok = (unsigned)s < (unsigned)c.pages && (unsigned)d < (unsigned)c.pages, late = false;
    for (int j0 = 0; j0 < count; j0 += 256) {
        __syncthreads();
        if (j0 + (int)threadIdx.x < count) tile[threadIdx.x] = dst[j0 + threadIdx.x];
        __syncthreads();
        for (int j = 0; j < min(256, count - j0); ++j) {
            late |= tile[j] == d && j0 + j > i;
            ok &= tile[j] != s || s == d;
        }
    }
    if (i >= count) return;
    if (!ok) kv_flag(c, Q3C_KV_BAD_PAGE);
    ws[i] = ok && !late && s != d ? s : -1;
}
__global__ void __launch_bounds__(256) kv_copy_kernel(const KvPieces pc, const int* __restrict__ src, const int* __restrict__ dst) {
    const int per = pc.layers * pc.per_layer, i = blockIdx.x / per, s = src[i];
    if (s >= 0) kv_copy_piece(pc, blockIdx.x - i * per, s, dst[i]);
}

// compact, first launch: the live pages behind the first `live` ones (sources, ascending) take the free ones before (destinations,
// ascending), so the two sets are disjoint and no page moves that need not.  ws: [0] pairs, [4 ..] pairs' sources, [4 + pages / 2 ..]
// their destinations, [4 + 2 (pages / 2) ..] where each page goes.
__global__ void __launch_bounds__(PLAN_T) kv_compact_plan_kernel(const KvView c, int* __restrict__ live, int* __restrict__ ws) {
    __shared__ int lds[17 + PLAN_K * 16];
    const int tid = threadIdx.x, half = c.pages / 2;
    int *src = ws + 4, *dst = src + half, *to = dst + half;
    for (int p = tid; p < c.pages; p += PLAN_T) to[p] = p;
    const int n = plan_pages(c, 0, c.pages, c.pages, lds, [](int r) { return r > 0; }, [](int, int) {});
    const int m = plan_pages(c, n, c.pages, half, lds, [](int r) { return r > 0; }, [&](int rank, int p) { src[rank] = p; });
    plan_pages(c, 0, n, m, lds, [](int r) { return r <= 0; }, [&](int rank, int p) { dst[rank] = p; });
    __syncthreads();
    for (int i = tid; i < m; i += PLAN_T) {
        const int s = src[i], d = dst[i];
        to[s] = d;
        c.refs[d] = c.refs[s];
        c.refs[s] = 0;
    }
    if (tid == 0) { ws[0] = m; *live = n; }
}
// compact, second launch: the first `table_blocks` blocks rewrite the table, the others copy pages
__global__ void __launch_bounds__(256) kv_compact_kernel(const KvView c, const KvPieces pc, int table_blocks, const int* __restrict__ ws) {
    const int half = c.pages / 2;
    const int *src = ws + 4, *dst = src + half, *to = dst + half;
    if ((int)blockIdx.x < table_blocks) {
        const long long n = (long long)c.rows * c.width;
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)table_blocks * 256) {
            const int p = c.table[i];
            if ((unsigned)p < (unsigned)c.pages) c.table[i] = to[p];
        }
        return;
    }
    const int per_pair = pc.layers * pc.per_layer;
    const long long n = (long long)ws[0] * per_pair;
    for (long long w = (int)blockIdx.x - table_blocks; w < n; w += (int)gridDim.x - table_blocks) {
        const int i = (int)(w / per_pair);
        kv_copy_piece(pc, (int)(w - (long long)i * per_pair), src[i], dst[i]);
    }
}

int lanes_shift(int dim, int per_lane = 8) {            // lanes of one head, rounded up to a power of two
    int s = 1;
    while ((per_lane << s) < dim) ++s;
    return s;
}

}  // namespace

hipError_t q3_launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
    const int d4 = a.c.dtype == Q3C_KV_INT4 ? a.c.dim : 0, units = a.q_heads + (d4 ? 0 : 2 * a.c.heads);
    // bf16: 16-byte accesses (runs of 8) where heads, halves and strides allow it, else 8-byte ones
    const auto wide = [](const KvStrided& x) { return x.ts % 8 == 0 && x.hs % 8 == 0 && (uintptr_t)x.p % 16 == 0; };
    const bool v8 = a.c.dtype != Q3C_KV_F32 && a.rot % 16 == 0 && wide(a.q) && (d4 || (wide(a.k) && wide(a.v)));
    const int sh = lanes_shift(a.c.dim, v8 ? 16 : 8), upw = 64 >> sh, runs = (units + upw - 1) / upw;
    int parts = runs;                       // waves of a token: few tokens are spread, many keep two runs of heads in flight per wave
    while (parts > 1 && (long long)a.b.tokens * parts > 4096 && (runs + parts - 1) / parts < 2) parts = (parts + 1) / 2;
    const int waves = parts + (d4 ? (2 * a.c.heads + 4 * M4 - 1) / (4 * M4) : 0);
    const unsigned blocks = (unsigned)(((long long)a.b.tokens * waves + 3) / 4);
    if (!blocks) return hipSuccess;
#define Q3_APPEND(T, D4)                                                                    \
    do {                                                                                    \
        if (v8) kv_append_kernel<T, 8, D4><<<blocks, 256, 0, s>>>(a, parts, waves, sh);     \
        else kv_append_kernel<T, 4, D4><<<blocks, 256, 0, s>>>(a, parts, waves, sh);        \
    } while (0)
    if (a.c.dtype == Q3C_KV_F32) kv_append_kernel<float, 4, 0><<<blocks, 256, 0, s>>>(a, parts, waves, sh);
    else if (!d4) Q3_APPEND(bf16, 0);
    else if (d4 == 64) Q3_APPEND(bf16, 64);
    else if (d4 == 128) Q3_APPEND(bf16, 128);
    else Q3_APPEND(bf16, 256);
#undef Q3_APPEND
    return hipGetLastError();
}

hipError_t q3_launch_kv_gather(const KvView& c, const KvBatch& b, int layer, void* k_out, void* v_out, int out_dtype, hipStream_t s) {
    const int sh = lanes_shift(c.dim), upw = 64 >> sh, runs = (2 * c.heads + upw - 1) / upw;
    int waves = runs;                       // of a token: few tokens are spread, many keep several heads in flight per wave
    while (waves > 1 && (long long)b.tokens * waves > 4096 && (runs + waves - 1) / waves < 4) waves = (waves + 1) / 2;
    const unsigned blocks = (unsigned)(((long long)b.tokens * waves + 3) / 4);
    if (!blocks) return hipSuccess;
#define Q3_GATHER(T, D4)                                                                                                       \
    (out_dtype == Q3_F32 ? kv_gather_kernel<T, float, D4><<<blocks, 256, 0, s>>>(c, b, layer, (float*)k_out, (float*)v_out, waves, sh) \
                         : kv_gather_kernel<T, bf16, D4><<<blocks, 256, 0, s>>>(c, b, layer, (bf16*)k_out, (bf16*)v_out, waves, sh))
    if (c.dtype == Q3C_KV_F32) Q3_GATHER(float, 0);
    else if (c.dtype == Q3C_KV_BF16) Q3_GATHER(bf16, 0);
    else if (c.dim == 64) Q3_GATHER(bf16, 64);
    else if (c.dim == 128) Q3_GATHER(bf16, 128);
    else Q3_GATHER(bf16, 256);
#undef Q3_GATHER
    return hipGetLastError();
}

hipError_t q3_launch_kv_reserve(const KvView& c, const KvBatch& b, hipStream_t s) {
    if (b.sequences > 0) kv_reserve_kernel<<<1, PLAN_T, 0, s>>>(c, b);
    return hipGetLastError();
}

hipError_t q3_launch_kv_release(const KvView& c, const int* rows, int count, int trim, int window, int sinks, hipStream_t s) {
    const int blocks = (c.width + 255) / 256;
    if (count > 0) kv_release_kernel<<<dim3(count, blocks < 4096 ? blocks : 4096), 256, 0, s>>>(c, rows, trim, window, sinks);
    return hipGetLastError();
}

hipError_t q3_launch_kv_fork(const KvView& c, const int* parents, const int* children, int count, int* ws, hipStream_t s) {
    if (count <= 0) return hipSuccess;
    const KvPieces pc = kv_pieces(c);
    kv_fork_plan_kernel<<<1, PLAN_T, 0, s>>>(c, parents, children, count, ws);
    kv_fork_kernel<<<(unsigned)count * (1 + pc.layers * pc.per_layer), 256, 0, s>>>(c, pc, parents, children, count, ws);
    return hipGetLastError();
}

hipError_t q3_launch_kv_copy(const KvView& c, const int* src, const int* dst, int count, int* ws, hipStream_t s) {
    if (count <= 0) return hipSuccess;
    const KvPieces pc = kv_pieces(c);
    kv_pairs_kernel<<<(count + 255) / 256, 256, 0, s>>>(c, src, dst, count, ws);
    kv_copy_kernel<<<(unsigned)count * (pc.layers * pc.per_layer), 256, 0, s>>>(pc, ws, dst);
    return hipGetLastError();
}

hipError_t q3_launch_kv_compact(const KvView& c, int* live, int* ws, hipStream_t s) {
    const KvPieces pc = kv_pieces(c);
    kv_compact_plan_kernel<<<1, PLAN_T, 0, s>>>(c, live, ws);
    const long long most = (long long)(c.pages / 2) * pc.layers * pc.per_layer;
    const int tb = (int)((((long long)c.rows * c.width + 255) / 256 < 64) ? ((long long)c.rows * c.width + 255) / 256 : 64);
    const int cb = (int)(most < 4096 ? most : 4096);          // persistent: how many pairs there are is known on the device only
    kv_compact_kernel<<<tb + cb, 256, 0, s>>>(c, pc, tb, ws);
    return hipGetLastError();
}
