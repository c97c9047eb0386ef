// What the kernels of the attention between two ragged sets of rows share: the arguments of a call, which rows a block works
// on, and how the long axis is split.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace hgc {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxDim = 128;
constexpr int kMaxCount = 0x7fffffff - 8192;  // rows of either set: a step past the end must not leave 32 bits
// Heads that share a key head are packed into the rows of a tile up to this many, so that keys and values are read once for all
// of them; beyond it every head has its own tiles.
constexpr int kMaxPack = 32;

// One call.  Rows of q, k and v are `row` and heads `head` elements apart, columns lie next to each other; every other tensor
// is dense.
struct Strided {
    const void *p;
    long long row, head;
};

struct Args {
    Strided q, k, v;
    const int *rs_q, *rs_k;        // [n_events + 1]
    const unsigned char *mask;     // [n_k], zero: no query sees the key; may be null
    const void *grad, *out;        // of the backward pass
    const void *out_rest;          // what the rounding of out left, or null
    void *rest;                    // of the forward pass: where that goes, or null
    const float2 *stats;           // [n_q, heads]: what the exponents of a row's weights are less by, and delta, the sum of out * grad
    const int *visible;            // [n_events], keys that can be seen, counted up to two
    float *lse;                    // [n_q, heads], natural logarithm of the sum of exp(scale * q.k)
    void *to, *to2;                // result: out, dq, or dk and dv
    float *part, *part2;           // the same of every part of a split, in float32
    float *part_lse;               // [splits, n_q, heads]
    // of half precision's backward pass: squared norms of the rows of grad, [n_q, heads], and the largest ones of the rows of grad and of v
    // that count in an event, [n_events, 2]
    const float *norms, *bounds;
    int *counter;                  // of the tiles that the blocks of the forward pass take
    unsigned *status;
    int n_q, n_k, n_events, heads, kv_heads, group, pack, dim, splits, alternate;  // alternate: of the forward pass on the tensor cores, two parts to each of the splits
    float scale, shift;            // shift: what `stats` is less by than the logarithms
};

// What a kernel before this one may have written is read after pdl_begin(), by a load that cannot move ahead of it as one of
// read-only data could.
template <typename T> __device__ __forceinline__ T fresh(const T *p) { return *const_cast<const volatile T *>(p); }

__device__ __forceinline__ int split_at(const int *rs, int i, int n) { return min(max(fresh(rs + i), 0), n); }

// The tiles of a ragged batch: event e owns the tile numbers from rs[e] / rows + e on, which leaves room for its last, partly
// filled tile whatever the lengths are, so that the host can size a grid (n / rows + n_events + 1) without reading the splits.
// What follows the last event is one more event, which has rows but no counterpart.
struct Tile {
    int event, begin, end;  // rows [begin, end); none: begin >= end
};

inline __host__ __device__ long long tile_count(int n, int rows, int n_events) { return (long long)n / rows + n_events + 1; }

// All 32 lanes of a warp call this; 32 events are looked at in a step.
__device__ __forceinline__ Tile find_tile(const int *rs, int n, int n_events, int rows, int tile)
{
    int lo = 0, hi = n_events + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5, at = lo + lane_id() * step;
        const bool before = at < hi && split_at(rs, at, n) / rows + at <= tile;
        const unsigned votes = __ballot_sync(0xffffffffu, before);
        const int ahead = max(votes == 0xffffffffu ? 32 : __ffs(~votes) - 1, 1);
        lo += (ahead - 1) * step;
        hi = min(lo + step, hi);
    }
    const int first = split_at(rs, lo, n), last = lo < n_events ? split_at(rs, lo + 1, n) : n;
    const long long begin = first + (long long)(tile - first / rows - lo) * rows;
    Tile t;
    t.event = lo;
    t.begin = begin < 0 || begin > last ? last : (int)begin;
    t.end = last - t.begin < rows ? last : t.begin + rows;  // no sum beyond 32 bits
    return t;
}

// The event of a row below `known`, the end of the last one: the last event that begins there or before.
__device__ __forceinline__ int event_of(const int *rs, int n, int n_events, int row)
{
    int lo = 0, hi = n_events;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (split_at(rs, mid, n) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same by the 32 lanes of a warp together.
__device__ __forceinline__ int event_of_warp(const int *rs, int n, int n_events, int row)
{
    int lo = 0, hi = n_events;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5, at = lo + lane_id() * step;
        const unsigned votes = __ballot_sync(0xffffffffu, at < hi && split_at(rs, at, n) <= row);
        lo += (max(votes == 0xffffffffu ? 32 : __ffs(~votes) - 1, 1) - 1) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// Steps [first, last) of part `s` of `n_parts` of a row of `steps`.
__device__ __forceinline__ int2 part_of(int steps, int s, int n_parts)
{
    const int each = (steps + n_parts - 1) / n_parts;
    return make_int2(min(s * each, steps), min((s + 1) * each, steps));
}

// Sets the status word: whether the splits ascend from zero to at most the number of rows.  Every access is clamped to the
// tensors whatever they hold.  One block of a call's first kernel does it, all of its threads together.
__device__ __forceinline__ void check_splits(const Args &a, int t, int threads)
{
    bool bad = false;
    for (int i = t; i <= a.n_events; i += threads) {
        const int q = fresh(a.rs_q + i), k = fresh(a.rs_k + i);
        bad |= q > (i < a.n_events ? fresh(a.rs_q + i + 1) : a.n_q) || k > (i < a.n_events ? fresh(a.rs_k + i + 1) : a.n_k);
        bad |= i == 0 && (q != 0 || k != 0);
    }
    const int any = __syncthreads_or(bad);
    if (t == 0) *a.status = any ? HGC_STATUS_ROW_SPLITS : 0u;
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A value, and what its rounding leaves where that is kept.
template <typename T> __device__ __forceinline__ void store_rounded(T *to, T *rest, float v)
{
    *to = from_float<T>(v);
    if (sizeof(T) == 2 && rest != nullptr) *rest = from_float<T>(v - to_float<T>(*to));
}

// keys of an event; none behind the last one
__device__ __forceinline__ int2 rows_of(const int *rs, int n, int n_events, int event)
{
    if (event >= n_events) return make_int2(0, 0);
    return make_int2(split_at(rs, event, n), split_at(rs, event + 1, n));
}

// A few queries per event (cross_attention_few.cu): rows of whole, aligned 16-byte vectors, up to eight rows of queries a block.
constexpr int kFewStep = 128;                        // keys that a split is a multiple of
int few_pack(int group);                             // heads of a block
int few_rows(int n_q, int n_events, int pack);       // rows of a block, or 0 where there are more than a few
bool few_takes(const Args &a, int rows, int dtype);
int few_forward(const Args &a, int rows, int dtype, cudaStream_t stream);

// The kernels on the tensor cores (cross_attention_mma.cu): 16-bit types, heads of whole 16-byte vectors, aligned rows.
bool mma_takes(const Args &a, int dtype);
constexpr int kMmaRows = 128;
inline __host__ __device__ int mma_keys(int dim) { return dim <= 64 ? 128 : 64; }  // keys of a step of the forward pass
constexpr int kMmaGradStep = 64;  // keys, or queries, of a step of the backward pass
int mma_forward(const Args &a, int dtype, cudaStream_t stream);
int mma_grad_queries(const Args &a, int dtype, cudaStream_t stream);
int mma_grad_keys(const Args &a, int dtype, cudaStream_t stream);
// Weights of the backward pass in half precision are held 2^14 times as large.
constexpr float kHalfShift = 14.f;

}  // namespace attn
}  // namespace hgc
