// Internal interface of the paged key/value cache (include/q3c.h, q3c_kv_*): what the entry points hand to the launchers, and the
// device helpers its kernels share.
#pragma once
#include "common.h"
#include "../../include/q3c.h"

struct KvView {
    int dtype;                          // q3c_kv_dtype
    int layers, pages, heads, ps_shift, dim, rows, width;   // page size = 1 << ps_shift; width = table entries of a row
    void *k, *v;                        // [layers][pages][heads][page][dim] (4 bits: [dim / 2] bytes a row)
    bf16 *ks, *vs;                      // 4 bits: steps [layers][pages][heads][page][dim / 32]
    int *table, *lens, *refs, *status;
};
// new tokens of a call: request i's are offsets[i] .. offsets[i+1] - 1 (null: token i alone), its last one at position lens[row] - 1.  An offset
// outside 0 .. tokens counts as the nearer end, in every kernel: reserve, append, gather and attend place a token alike.
struct KvBatch { const int* rows; const int* offsets; int sequences, tokens; };
struct KvStrided { const void* p; long long ts, hs; };          // [token][head][dim], strides in elements, dim contiguous

struct KvAppendArgs {
    KvView c; KvBatch b; int layer;
    KvStrided q, k, v;
    int q_heads;
    const float *qw, *kw, *cos_t, *sin_t;                       // norm weights [dim] or null, tables [positions][rot / 2]
    int rot;
    float eps, inv_dim;
    void* q_out;                                                // [tokens][q_heads][dim]
};
struct KvAttendArgs {
    KvView c; KvBatch b; int layer;
    KvStrided q;
    int q_heads, group, window, sinks;
    float scale_log2e;
    void* out;                                                  // [tokens][q_heads][dim]
    int most;                                                   // chunks that a row can see
    int splits, share;                                          // shares of a tile's key chunks: most there can be, chunks of one
    float* ws;
};
hipError_t q3_launch_kv_append(const KvAppendArgs& a, hipStream_t s);
hipError_t q3_launch_kv_gather(const KvView& c, const KvBatch& b, int layer, void* k_out, void* v_out, int out_dtype, hipStream_t s);
hipError_t q3_launch_kv_reserve(const KvView& c, const KvBatch& b, hipStream_t s);
hipError_t q3_launch_kv_release(const KvView& c, const int* rows, int count, int trim, int window, int sinks, hipStream_t s);
hipError_t q3_launch_kv_fork(const KvView& c, const int* parents, const int* children, int count, int* ws, hipStream_t s);
hipError_t q3_launch_kv_copy(const KvView& c, const int* src, const int* dst, int count, int* ws, hipStream_t s);
hipError_t q3_launch_kv_compact(const KvView& c, int* live, int* ws, hipStream_t s);
struct KvSplit { int splits, share, most; };
KvSplit q3_kv_attend_split(const KvView& c, int tokens, int sequences, int q_heads, bool ragged, int window, int sinks, int max_len);
size_t q3_kv_attend_ws(const KvView& c, int tokens, int sequences, int q_heads, bool ragged, int splits);
hipError_t q3_launch_kv_attend(const KvAttendArgs& a, hipStream_t s);

#ifdef __HIPCC__
// The request that token t belongs to = how many of offsets[1 .. n] are <= t.  Counted 64 entries at a time by the lanes of a
// wave (t uniform): independent loads where a bisection would wait for log2(n) dependent ones.
__device__ __forceinline__ int kv_find(const int* __restrict__ offsets, int n, int t, int lane) {
    int b = 0;
    for (int i = 0; i < n; i += 64) b += __popcll(__ballot(i + lane < n && offsets[min(i + lane, n - 1) + 1] <= t));
    return b;
}
// The cache position of new token t (wave-uniform); -1: it lies before the first request or behind the last, -2: bad row, or a position outside the row's
// table.  `seq`, `row`: its request and table row.
__device__ __forceinline__ int kv_position(const KvView& c, const KvBatch& b, int t, int lane, int& seq, int& row) {
    int back = 1;
    seq = t;
    if (b.offsets) {
        seq = kv_find(b.offsets, b.sequences, t, lane);
        if (seq >= b.sequences || (seq == 0 && t < b.offsets[0])) return -1;
        back = min(b.offsets[seq + 1], b.tokens) - t;
        if (back < 1) return -2;                                // offsets that do not ascend
    }
    row = b.rows[seq];
    if (row < 0 || row >= c.rows) return -2;
    const long long pos = (long long)c.lens[row] - back;
    return pos < 0 || pos >= ((long long)c.width << c.ps_shift) ? -2 : (int)pos;
}
// Whether the call's offsets end behind its tokens; true for its last token alone, whose wave reports it.
__device__ __forceinline__ bool kv_ends_behind(const KvBatch& b, int t) { return b.offsets && t == b.tokens - 1 && b.offsets[b.sequences] > b.tokens; }
#endif
