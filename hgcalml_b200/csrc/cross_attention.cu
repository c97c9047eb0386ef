// Attention between two ragged sets of rows of the same events, forward and backward: products in float32 on the tensor cores,
// in parts, for every type, width and stride, and the C entries.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / l_i,  s_ij = scale q_i.k_j over the keys j of i's event that can be seen
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - delta_i),  delta_i = do_i.o_i,  dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i
//
// A row without keys has o = 0, and -inf for the logarithm of its sum.  Gradients of shared key heads are summed inside the
// kernel and parts of a split are joined in their order, so results do not change from run to run (atomics take the largest of some
// norms, and the next tile, whose order changes none).
#include "cross_attention.cuh"
#include "mma_device.cuh"

namespace hgc {
namespace attn {
namespace {

constexpr int kRows = 64;        // rows and columns of a tile
constexpr int kThreads = 256;    // four times two warps: a warp has 16 rows and 32 columns of a tile of scores
constexpr int kWarpRows = 16, kWarpColumns = 32, kBlocks = kWarpColumns / 8;  // of 8 columns, which one product has

// Products on the tensor cores, of which this form takes operands of 11 bits: x = big + small, both of 11 bits, and a product is
// big big + big small + small big, off by what is left of either, 2^-21, and by small small, 2^-22.  Tensor cores cut off what an
// addition leaves, so the small products have a sum of their own, and sums are taken on from there with rounding, once a step.
// On the CUDA cores a tile of 4 x 4 per thread waited for shared memory half of the time (7 events of some 16k rows on 2.6k, 22 columns:
// 4661 us, here 2868; a training step on three of 7k on 2k, 32 columns: 4596, here 2739), and was less exact.  What bounds it: sixteen
// warps, for which there are registers, with ten instructions to a product; the tensor cores are half busy.
// 16-bit values are operands as they are (`EXACT`).
//
// A lane of a warp has the rows g and g + 8, g = lane / 4, and of 8 columns those from 2 (lane % 4) on.  What one product leaves is an
// operand of the next one where it is: the order of summed rows is free, so lane t takes the rows 2 t and 2 t + 1 of the other operand.
__device__ __forceinline__ void product(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2])
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <bool EXACT> __device__ __forceinline__ void in_two(float x, unsigned &big, unsigned &small)
{
    if constexpr (EXACT) {
        big = __float_as_uint(x);
    } else {
        big = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
        small = __float_as_uint(x - __uint_as_float(big)) & 0xffffe000u;
    }
}

// Rows of `DP` floats, 4 more apart: neither kind of operand meets a bank twice.
template <int DP> constexpr int kPitch = DP + 4;

// s[n][i] = row of a . row of b, for 16 rows of a and 32 of b.
template <int DP, bool EXACT>
__device__ __forceinline__ void dots(float (&s)[kBlocks][4], const float *__restrict__ a, const float *__restrict__ b, int dim)
{
    constexpr int P = kPitch<DP>;
    const int at = (lane_id() >> 2) * P + (lane_id() & 3);
    float rest[kBlocks][4];
#pragma unroll
    for (int n = 0; n < kBlocks; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] = rest[n][i] = 0.f;
#pragma unroll
    for (int d = 0; d < DP; d += 8) {
        if (d >= dim) break;
        unsigned a_big[4], a_small[4];
#pragma unroll
        for (int i = 0; i < 4; i++) in_two<EXACT>(a[at + (i & 1) * 8 * P + d + (i >> 1) * 4], a_big[i], a_small[i]);
#pragma unroll
        for (int n = 0; n < kBlocks; n++) {
            unsigned b_big[2], b_small[2];
#pragma unroll
            for (int i = 0; i < 2; i++) in_two<EXACT>(b[at + n * 8 * P + d + i * 4], b_big[i], b_small[i]);
            if constexpr (!EXACT) {
                product(rest[n], a_small, b_big);
                product(rest[n], a_big, b_small);
            }
            product(s[n], a_big, b_big);
        }
    }
    if constexpr (!EXACT) {
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] += rest[n][i];
    }
}

// acc[n][i] += sum over the 32 rows of b, weighted by w as dots() leaves it.
template <int DP, bool EXACT>
__device__ __forceinline__ void weighted_rows(float (&acc)[DP / 8][4], const float (&w)[kBlocks][4], const float *__restrict__ b, int dim)
{
    constexpr int P = kPitch<DP>;
    const int at = 2 * (lane_id() & 3) * P + (lane_id() >> 2);
    unsigned w_big[kBlocks][4], w_small[kBlocks][4];
#pragma unroll
    for (int k = 0; k < kBlocks; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) in_two<false>(w[k][(i & 1) * 2 + (i >> 1)], w_big[k][i], w_small[k][i]);
#pragma unroll
    for (int n = 0; n < DP / 8; n++) {
        if (8 * n >= dim) break;
        float sum[4] = {}, rest[4] = {};
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            unsigned b_big[2], b_small[2];
#pragma unroll
            for (int i = 0; i < 2; i++) in_two<EXACT>(b[at + (8 * k + i) * P + 8 * n], b_big[i], b_small[i]);
            product(rest, w_small[k], b_big);
            if constexpr (!EXACT) product(rest, w_big[k], b_small);
            product(sum, w_big[k], b_big);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += sum[i] + rest[i];
    }
}
// The warps of the second 32 columns leave their sums in shared memory, after a barrier, the others have them added to theirs.
template <int DP> __device__ __forceinline__ void leave(float *__restrict__ to, const float (&acc)[DP / 8][4])
{
    float *at = to + (lane_id() >> 2) * kPitch<DP> + 2 * (lane_id() & 3);
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i += 2) *reinterpret_cast<float2 *>(at + i * 4 * kPitch<DP> + 8 * n) = make_float2(acc[n][i], acc[n][i + 1]);
}
template <int DP> __device__ __forceinline__ void add(float (&acc)[DP / 8][4], const float *__restrict__ from, const float (&mine)[2], const float (&theirs)[2])
{
    const float *at = from + (lane_id() >> 2) * kPitch<DP> + 2 * (lane_id() & 3);
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = acc[n][i] * mine[i >> 1] + at[(i >> 1) * 8 * kPitch<DP> + 8 * n + (i & 1)] * theirs[i >> 1];
}
// Row `row` (0, or 1: 8 further) of a warp's results, times `factor`, to `to`.
template <int DP, typename T>
__device__ __forceinline__ void store_row(T *__restrict__ to, const float (&acc)[DP / 8][4], int row, float factor, int dim, T *__restrict__ rest = nullptr)
{
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int d = 8 * n + 2 * (lane_id() & 3) + i;
            if (d < dim) store_rounded(to + d, rest == nullptr ? rest : rest + d, acc[n][2 * row + i] * factor);
        }
}

// Rows of one head as floats; what is not there, and the keys that cannot be seen, are zeros, whatever the memory holds: a weight of
// zero would not make up for an infinity.  Copies are in pieces of 16, 8 or 4 bytes as the rows allow, single values in 16 bits.
// In float32 they are asynchronous (copied() waits for all but the last `ahead` groups); other types are converted on their way.
template <typename T> __device__ __forceinline__ int piece_of(const Strided &s, int dim)
{
    constexpr unsigned long long kSize = sizeof(T);
    const unsigned long long all = reinterpret_cast<unsigned long long>(s.p) | s.row * kSize | s.head * kSize | dim * kSize;
    return (all & 15u) == 0 ? 16 / sizeof(T) : kSize == 4 && (all & 7u) == 0 ? 2 : 1;
}
template <int N> __device__ __forceinline__ void copy_async(float *dst, const float *src, bool in)  // zeros where not `in`
{
    const unsigned to = (unsigned)__cvta_generic_to_shared(dst);
    if constexpr (N == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(src), "r"(in ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" :: "r"(to), "l"(src), "r"(in ? 4 * N : 0), "n"(4 * N) : "memory");
}
template <int AHEAD> __device__ __forceinline__ void copied() { asm volatile("cp.async.wait_group %0;" :: "n"(AHEAD) : "memory"); }
__device__ __forceinline__ void end_of_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// `place(r)`: where row r begins, or a negative number
template <typename T, int DP, int N, typename Place>
__device__ __forceinline__ void copy_rows(float *__restrict__ dst, const T *__restrict__ p, int dim, Place place)
{
    constexpr int W = DP / N;
#pragma unroll 4
    for (int i = threadIdx.x; i < kRows * W; i += kThreads) {
        const int r = i / W, d = i % W * N;
        const long long at = place(r);
        const bool in = at >= 0 && d < dim;
        if constexpr (sizeof(T) == 4) {
            copy_async<N>(dst + r * kPitch<DP> + d, p + (in ? at + d : 0), in);
        } else if constexpr (N == 8) {
            const uint4 v = in ? *reinterpret_cast<const uint4 *>(p + at + d) : make_uint4(0, 0, 0, 0);
            const float2 f[4] = {mma::unpack2<T>(v.x), mma::unpack2<T>(v.y), mma::unpack2<T>(v.z), mma::unpack2<T>(v.w)};
            float4 *to = reinterpret_cast<float4 *>(dst + r * kPitch<DP> + d);
            to[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            to[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
        } else {
            dst[r * kPitch<DP> + d] = in ? to_float(p[at + d]) : 0.f;
        }
    }
}
template <typename T, int DP, typename Place>
__device__ __forceinline__ void load_rows(float *__restrict__ dst, const Strided &s, int piece, int dim, Place place)
{
    const T *p = static_cast<const T *>(s.p);
    if constexpr (sizeof(T) == 4) {
        if (piece == 4) return copy_rows<T, DP, 4>(dst, p, dim, place);
        if (piece == 2) return copy_rows<T, DP, 2>(dst, p, dim, place);
    } else {
        if (piece == 8) return copy_rows<T, DP, 8>(dst, p, dim, place);
    }
    copy_rows<T, DP, 1>(dst, p, dim, place);
}
// keys that can be seen, of those of a step
__device__ __forceinline__ void load_seen(unsigned char *seen, const unsigned char *mask, int begin, int n)
{
    if (threadIdx.x < kRows) seen[threadIdx.x] = (int)threadIdx.x < n && (mask == nullptr || mask[begin + threadIdx.x] != 0);
}
template <typename T, int DP>
__device__ __forceinline__ void load_keys(float *__restrict__ dst, const Strided &s, int piece, int head, int begin, int dim, const unsigned char *seen)
{
    load_rows<T, DP>(dst, s, piece, dim, [&](int r) { return seen[r] ? (long long)(begin + r) * s.row + (long long)head * s.head : -1ll; });
}
// row r of a tile of queries is head r % pack of token r / pack
template <typename T, int DP>
__device__ __forceinline__ void load_queries(float *__restrict__ dst, const Strided &s, int piece, int head0, int begin, int n, int pack, int dim)
{
    load_rows<T, DP>(dst, s, piece, dim, [&](int r) {
        return r < n ? (long long)(begin + r / pack) * s.row + (long long)(head0 + r % pack) * s.head : -1ll;
    });
}
// The next step's rows are on their way during this one; the widest heads have no room for that, but a second block has.
template <int DP> constexpr int kStages = DP <= 64 ? 2 : 1;

// The block's tile, found by the first warp; blocks of one call that have nothing to do leave here.
__device__ __forceinline__ Tile block_tile(const int *rs, int n, int n_events, int rows)
{
    __shared__ Tile s_tile;
    if (threadIdx.x < 32) {
        const Tile t = find_tile(rs, n, n_events, rows, blockIdx.x);
        if (threadIdx.x == 0) s_tile = t;
    }
    __syncthreads();
    return s_tile;
}

// ------------------------------------------------------------------------------------------------------------- forward
// A block takes a tile of queries (with the heads that share a key head) through the keys of its event, 64 at a time, with the
// running maximum and sum of every row.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const __grid_constant__ Args a)
{
    pdl_begin();
    constexpr int P = kPitch<DP>, S = kStages<DP>;
    constexpr bool kExact = sizeof(T) == 2;
    extern __shared__ __align__(16) float s_mem[];
    float *s_q = s_mem, *s_k = s_q + kRows * P, *s_v = s_k + S * kRows * P;
    __shared__ unsigned char s_seen_all[S][kRows];
    const int t = threadIdx.x, row0 = (t >> 5) % 4 * kWarpRows, column0 = (t >> 7) * kWarpColumns;
    const int tokens = kRows / a.pack, head0 = blockIdx.y * a.pack, kv = head0 / a.group;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_splits(a, t, kThreads);
    const Tile tile = block_tile(a.rs_q, a.n_q, a.n_events, tokens);
    if (tile.begin >= tile.end) return;
    const int n_rows = (tile.end - tile.begin) * a.pack;
    const int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    const int2 part = part_of(max(0, (keys.y - keys.x + kRows - 1) / kRows), blockIdx.z, a.splits);
    load_queries<T, DP>(s_q, a.q, piece_of<T>(a.q, a.dim), head0, tile.begin, n_rows, a.pack, a.dim);
    end_of_copies();  // a group of their own: with no step after it, they are waited for at the end all the same
    const int piece_k = piece_of<T>(a.k, a.dim), piece_v = piece_of<T>(a.v, a.dim);
    const auto load = [&](int step) {  // with a barrier inside
        const int at = step % S, k0 = keys.x + step * kRows;
        if (step < part.y) load_seen(s_seen_all[at], a.mask, k0, min(kRows, keys.y - k0));
        __syncthreads();
        if (step < part.y) {
            load_keys<T, DP>(s_k + at * kRows * P, a.k, piece_k, kv, k0, a.dim, s_seen_all[at]);
            load_keys<T, DP>(s_v + at * kRows * P, a.v, piece_v, kv, k0, a.dim, s_seen_all[at]);
        }
        end_of_copies();
    };
    if (S > 1) load(part.x);
    const float c = a.scale * kLog2e;
    float o[DP / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
    for (int step = part.x; step < part.y; step++) {
        __syncthreads();  // the buffers that are filled now have been read
        load(step + S - 1);
        copied<S - 1>();
        __syncthreads();
        const float *k_now = s_k + step % S * kRows * P, *v_now = s_v + step % S * kRows * P;
        const unsigned char *s_seen = s_seen_all[step % S] + column0 + 2 * (lane_id() & 3);
        float s[kBlocks][4];
        dots<DP, kExact>(s, s_q + row0 * P, k_now + column0 * P, a.dim);
#pragma unroll
        for (int r = 0; r < 2; r++) {
            float top = m[r];
#pragma unroll
            for (int n = 0; n < kBlocks; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    if (!s_seen[8 * n + i]) s[n][2 * r + i] = -INFINITY;
                    top = fmaxf(top, s[n][2 * r + i]);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float base = top == -INFINITY ? 0.f : top;
            if (__any_sync(0xffffffffu, top > m[r])) {
                const float shrink = mma::exp2_fast((m[r] - base) * c);
                l[r] *= shrink;  // of this lane's columns
#pragma unroll
                for (int n = 0; n < DP / 8; n++) {
                    o[n][2 * r] *= shrink;
                    o[n][2 * r + 1] *= shrink;
                }
                m[r] = top;
            }
#pragma unroll
            for (int n = 0; n < kBlocks; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    s[n][2 * r + i] = mma::exp2_fast((s[n][2 * r + i] - base) * c);
                    l[r] += s[n][2 * r + i];
                }
        }
        weighted_rows<DP, kExact>(o, s, v_now + column0 * P, a.dim);
    }
    // the two times 32 columns
    __shared__ float2 s_stats[kRows];
    copied<0>();
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; r++) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (column0 > 0 && (lane_id() & 3) == 0) s_stats[row0 + (lane_id() >> 2) + 8 * r] = make_float2(m[r], l[r]);
    }
    if (column0 > 0) leave<DP>(s_q + row0 * P, o);
    __syncthreads();
    if (column0 > 0) return;
    float mine[2], theirs[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const float2 other = s_stats[row0 + (lane_id() >> 2) + 8 * r];
        const float top = fmaxf(m[r], other.x), base = top == -INFINITY ? 0.f : top;
        mine[r] = exp2f((m[r] - base) * c);
        theirs[r] = exp2f((other.x - base) * c);
        l[r] = l[r] * mine[r] + other.y * theirs[r];
        m[r] = top;
    }
    add<DP>(o, s_q + row0 * P, mine, theirs);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = row0 + (lane_id() >> 2) + 8 * i;
        if (r >= n_rows) continue;
        const long long row = (long long)(tile.begin + r / a.pack) * a.heads + head0 + r % a.pack;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        float *lse_to = a.splits > 1 ? a.part_lse + (long long)blockIdx.z * a.n_q * a.heads : a.lse;
        if ((lane_id() & 3) == 0) lse_to[row] = l[i] == 0.f ? -INFINITY : m[i] * a.scale + logf(l[i]);
        if (a.splits > 1) store_row<DP>(a.part + ((long long)blockIdx.z * a.n_q * a.heads + row) * a.dim, o, i, inv, a.dim);
        else store_row<DP>(static_cast<T *>(a.to) + row * a.dim, o, i, inv, a.dim, a.rest == nullptr ? nullptr : static_cast<T *>(a.rest) + row * a.dim);
    }
}

// Joins the parts of a row: every part holds its own softmax and the logarithm of its sum.
constexpr int kMaxParts = 128;
template <typename T>
__global__ void __launch_bounds__(256)
join_forward_kernel(const float *__restrict__ part, const float *__restrict__ part_lse, T *__restrict__ out, T *__restrict__ rest,
                    float *__restrict__ lse, long long n_rows, int dim, int splits)
{
    pdl_begin();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= n_rows) return;
    // a lane has every 32nd part's logarithm
    constexpr int kEach = kMaxParts / 32;
    float lse_of[kEach], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int s = 32 * i + lane_id();
        lse_of[i] = s < splits ? part_lse[s * n_rows + row] : -INFINITY;
        top = fmaxf(top, lse_of[i]);
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        lse_of[i] = exp2f((lse_of[i] - base) * kLog2e);
        sum += lse_of[i];
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int d0 = 0; d0 < dim; d0 += 32) {
        const int d = d0 + lane_id();
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
#pragma unroll 8
            for (int s = 0; s < min(32, splits - 32 * i); s++) {
                const float w = __shfl_sync(0xffffffffu, lse_of[i], s);
                // parts without weight were not written
                const float v = d < dim ? part[((32ll * i + s) * n_rows + row) * dim + d] : 0.f;
                o = fmaf(w, w == 0.f ? 0.f : v, o);
            }
        }
        if (d < dim) store_rounded(out + row * dim + d, rest == nullptr ? rest : rest + row * dim + d, o * inv);
    }
    if (lane_id() == 0) lse[row] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// ------------------------------------------------------------------------------------------------------------ backward
// What both gradients go by.  The first `n_count` blocks: the keys of an event that can be seen, counted up to two; with one key
// the weights do not depend on the scores, so the gradients of q and k are zero and not what is left of two sums that cancel.
// The next `n_rows` blocks, for every row of the queries: what its exponents are less by (log2 of its sum, less `shift`; infinity
// without keys) and delta.  With `bounds`: the squared norms of the rows of grad there, and of every event the largest one that
// counts of these, and of the rows of v in the blocks that follow.
constexpr int kRowsALane = 4;
template <typename T>
__global__ void __launch_bounds__(kThreads)
prepare_backward_kernel(const __grid_constant__ Args a, float2 *__restrict__ stats, int *__restrict__ visible, float *__restrict__ norms,
                        float *__restrict__ bounds, float shift, int n_count, int n_rows, int lanes_log2)
{
    pdl_begin();
    const int t = threadIdx.x;
    int block = blockIdx.x;
    if (block < n_count) {
        const int e = block;
        if (e == 0) check_splits(a, t, kThreads);
        if (e >= a.n_events) return;
        const int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, e);
        int n = a.mask == nullptr ? max(0, keys.y - keys.x) : 0;
        for (int base = keys.x; a.mask != nullptr && base < keys.y && n < 2; base += kThreads)
            n += __syncthreads_count(base + t < keys.y && a.mask[base + t] != 0);
        if (t == 0) visible[e] = min(n, 2);
        return;
    }
    block -= n_count;
    float norm = 0.f;
    // 2^lanes_log2 lanes have a row, 16 bytes each, or all 32 of them single columns; four rows a lane are on their way at a time
    const bool whole = lanes_log2 >= 0;
    const int lanes = whole ? 1 << lanes_log2 : 32, lane = t & (lanes - 1), subs = kThreads / lanes;
    constexpr int V = 16 / sizeof(T);
    struct alignas(16) Vec { T v[V]; };
    const bool of_queries = block < n_rows;
    const long long all = of_queries ? (long long)a.n_q * a.heads : (long long)a.n_k * a.kv_heads;
    const long long first = (long long)(of_queries ? block : block - n_rows) * (subs * kRowsALane) + t / lanes;
    const int known = of_queries ? split_at(a.rs_q, a.n_events, a.n_q) : split_at(a.rs_k, a.n_events, a.n_k);  // rows of some event
    const int *__restrict__ rs = of_queries ? a.rs_q : a.rs_k;
    const int n = of_queries ? a.n_q : a.n_k, per_row = of_queries ? a.heads : a.kv_heads;
    __shared__ int s_event;  // of all of the block's rows, or -1
    if (bounds != nullptr && t < 32) {
        const long long begin = (long long)(of_queries ? block : block - n_rows) * (subs * kRowsALane), end = min(begin + subs * kRowsALane, all);
        const int event = event_of_warp(rs, n, a.n_events, (int)(begin / per_row));
        if (t == 0) s_event = event + 1 >= a.n_events || (end - 1) / per_row < split_at(rs, event + 1, n) ? event : -1;
    }
    const T *__restrict__ out = static_cast<const T *>(a.out), *__restrict__ rest = static_cast<const T *>(a.out_rest),
            *__restrict__ grad = static_cast<const T *>(a.grad);
    float sum[kRowsALane], square[kRowsALane];
    if (whole) {
        Vec x[kRowsALane], y[kRowsALane], z[kRowsALane];
#pragma unroll
        for (int i = 0; i < kRowsALane; i++) {
            const long long row = first + (long long)i * subs;
            const bool in = row < all && lane * V < a.dim;
            x[i] = y[i] = z[i] = Vec{};
            if (in && of_queries) {
                x[i] = *reinterpret_cast<const Vec *>(out + row * a.dim + lane * V);
                if (sizeof(T) == 2 && rest != nullptr) z[i] = *reinterpret_cast<const Vec *>(rest + row * a.dim + lane * V);
                y[i] = *reinterpret_cast<const Vec *>(grad + row * a.dim + lane * V);
            } else if (in) {
                const int key = (int)(row / a.kv_heads);
                y[i] = *reinterpret_cast<const Vec *>(static_cast<const T *>(a.v.p) + key * a.v.row + (row - (long long)key * a.kv_heads) * a.v.head + lane * V);
            }
        }
#pragma unroll
        for (int i = 0; i < kRowsALane; i++) {
            sum[i] = square[i] = 0.f;
#pragma unroll
            for (int d = 0; d < V; d++) {
                const float g = to_float(y[i].v[d]);
                sum[i] = fmaf(to_float(x[i].v[d]) + to_float(z[i].v[d]), g, sum[i]);
                square[i] = fmaf(g, g, square[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRowsALane; i++) {
            const long long row = first + (long long)i * subs;
            sum[i] = square[i] = 0.f;
            for (int d = lane; d < a.dim && row < all; d += 32) {
                const int key = of_queries ? 0 : (int)(row / a.kv_heads);
                const float g = of_queries ? to_float(grad[row * a.dim + d])
                                           : to_float(static_cast<const T *>(a.v.p)[key * a.v.row + (row - (long long)key * a.kv_heads) * a.v.head + d]);
                if (of_queries) sum[i] = fmaf(to_float(out[row * a.dim + d]) + (rest == nullptr ? 0.f : to_float(rest[row * a.dim + d])), g, sum[i]);
                square[i] = fmaf(g, g, square[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kRowsALane; i++) {
        const long long row = first + (long long)i * subs;
        for (int w = lanes >> 1; w > 0; w >>= 1) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], w);
            square[i] += __shfl_xor_sync(0xffffffffu, square[i], w);
        }
        if (row >= all) continue;
        if (of_queries && lane == 0) {
            const float lse = a.lse[row];
            stats[row] = make_float2(lse == -INFINITY ? INFINITY : lse * kLog2e - shift, sum[i]);
            if (bounds != nullptr) norms[row] = square[i];
        }
    }
    if (bounds == nullptr) return;
    __syncthreads();
    // Norms are not negative, so their bits are in the order of their values: the largest one does not depend on the order of the blocks.
    // Rows behind the last event, and masked keys, are of no one's concern.
    const bool one_event = s_event >= 0;
#pragma unroll
    for (int i = 0; i < kRowsALane; i++) {
        const long long row = first + (long long)i * subs, token = row / per_row;
        if (row >= all || token >= known || (!of_queries && a.mask != nullptr && fresh(a.mask + token) == 0)) continue;
        if (one_event) norm = fmaxf(norm, square[i]);
        else if (lane == 0 && square[i] > 0.f)
            atomicMax(reinterpret_cast<unsigned *>(bounds) + 2 * event_of(rs, n, a.n_events, (int)token) + (of_queries ? 0 : 1), __float_as_uint(square[i]));
    }
    if (!one_event) return;
    __shared__ float s_norm[kThreads / 32];
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) norm = fmaxf(norm, __shfl_xor_sync(0xffffffffu, norm, w));
    if (lane_id() == 0) s_norm[t >> 5] = norm;
    __syncthreads();
    if (t == 0) {
        for (int i = 1; i < kThreads / 32; i++) norm = fmaxf(norm, s_norm[i]);
        if (norm > 0.f) atomicMax(reinterpret_cast<unsigned *>(bounds) + 2 * s_event + (of_queries ? 0 : 1), __float_as_uint(norm));
    }
}

// dq of a tile of queries: the keys of the event pass by once more.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads)
grad_queries_kernel(const __grid_constant__ Args a)
{
    pdl_begin();
    constexpr int P = kPitch<DP>, S = kStages<DP>;
    constexpr bool kExact = sizeof(T) == 2;
    extern __shared__ __align__(16) float s_mem[];
    float *s_q = s_mem, *s_g = s_q + kRows * P, *s_k = s_g + kRows * P, *s_v = s_k + S * kRows * P;
    __shared__ unsigned char s_seen_all[S][kRows];
    const int t = threadIdx.x, row0 = (t >> 5) % 4 * kWarpRows, column0 = (t >> 7) * kWarpColumns;
    const int tokens = kRows / a.pack, head0 = blockIdx.y * a.pack, kv = head0 / a.group;
    const Tile tile = block_tile(a.rs_q, a.n_q, a.n_events, tokens);
    if (tile.begin >= tile.end) return;
    const int n_rows = (tile.end - tile.begin) * a.pack;
    int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    if (tile.event < a.n_events && a.visible[tile.event] < 2) keys.y = keys.x;
    const int2 part = part_of(max(0, (keys.y - keys.x + kRows - 1) / kRows), blockIdx.z, a.splits);
    const Strided grad{a.grad, (long long)a.heads * a.dim, a.dim};
    load_queries<T, DP>(s_q, a.q, piece_of<T>(a.q, a.dim), head0, tile.begin, n_rows, a.pack, a.dim);
    load_queries<T, DP>(s_g, grad, piece_of<T>(grad, a.dim), head0, tile.begin, n_rows, a.pack, a.dim);
    end_of_copies();
    const int piece_k = piece_of<T>(a.k, a.dim), piece_v = piece_of<T>(a.v, a.dim);
    const auto load = [&](int step) {  // with a barrier inside
        const int at = step % S, k0 = keys.x + step * kRows;
        if (step < part.y) load_seen(s_seen_all[at], a.mask, k0, min(kRows, keys.y - k0));
        __syncthreads();
        if (step < part.y) {
            load_keys<T, DP>(s_k + at * kRows * P, a.k, piece_k, kv, k0, a.dim, s_seen_all[at]);
            load_keys<T, DP>(s_v + at * kRows * P, a.v, piece_v, kv, k0, a.dim, s_seen_all[at]);
        }
        end_of_copies();
    };
    if (S > 1) load(part.x);
    const float c = a.scale * kLog2e;
    float dq[DP / 8][4] = {}, lse[2], delta[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = row0 + (lane_id() >> 2) + 8 * i;
        const long long row = (long long)(tile.begin + r / a.pack) * a.heads + head0 + r % a.pack;
        const float2 stat = r < n_rows ? a.stats[row] : make_float2(INFINITY, 0.f);
        lse[i] = stat.x + a.shift;
        delta[i] = stat.y;
    }
    for (int step = part.x; step < part.y; step++) {
        __syncthreads();  // the buffers that are filled now have been read
        load(step + S - 1);
        copied<S - 1>();
        __syncthreads();
        const float *k_now = s_k + step % S * kRows * P + column0 * P, *v_now = s_v + step % S * kRows * P + column0 * P;
        const unsigned char *s_seen = s_seen_all[step % S] + column0 + 2 * (lane_id() & 3);
        float s[kBlocks][4], dp[kBlocks][4];
        dots<DP, kExact>(s, s_q + row0 * P, k_now, a.dim);
        dots<DP, kExact>(dp, s_g + row0 * P, v_now, a.dim);
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[n][i] = s_seen[8 * n + (i & 1)] ? mma::exp2_fast(fmaf(s[n][i], c, -lse[i >> 1])) * (dp[n][i] - delta[i >> 1]) : 0.f;
        weighted_rows<DP, kExact>(dq, s, k_now, a.dim);
    }
    copied<0>();
    __syncthreads();
    if (column0 > 0) leave<DP>(s_k + row0 * P, dq);
    __syncthreads();
    if (column0 > 0) return;
    const float one[2] = {1.f, 1.f};
    add<DP>(dq, s_k + row0 * P, one, one);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = row0 + (lane_id() >> 2) + 8 * i;
        if (r >= n_rows) continue;
        const long long row = (long long)(tile.begin + r / a.pack) * a.heads + head0 + r % a.pack;
        if (a.splits > 1) store_row<DP>(a.part + ((long long)blockIdx.z * a.n_q * a.heads + row) * a.dim, dq, i, a.scale, a.dim);
        else store_row<DP>(static_cast<T *>(a.to) + row * a.dim, dq, i, a.scale, a.dim);
    }
}

// dk and dv of a tile of keys: the queries of the event pass by, with all heads that share the key head.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads)
grad_keys_kernel(const __grid_constant__ Args a)
{
    pdl_begin();
    constexpr int P = kPitch<DP>, S = kStages<DP>;
    constexpr bool kExact = sizeof(T) == 2;
    extern __shared__ __align__(16) float s_mem[];
    float *s_q = s_mem, *s_g = s_q + S * kRows * P, *s_k = s_g + S * kRows * P, *s_v = s_k + kRows * P;
    __shared__ float2 s_stats_all[S][kRows];
    __shared__ unsigned char s_seen[kRows];
    const int t = threadIdx.x, row0 = (t >> 5) % 4 * kWarpRows, column0 = (t >> 7) * kWarpColumns, kv = blockIdx.y;
    const Tile tile = block_tile(a.rs_k, a.n_k, a.n_events, kRows);
    if (tile.begin >= tile.end) return;
    const int n_keys = tile.end - tile.begin, tokens = kRows / a.pack;
    const int2 queries = rows_of(a.rs_q, a.n_q, a.n_events, tile.event);
    const int blocks = max(0, (queries.y - queries.x + tokens - 1) / tokens), packs = a.group / a.pack;
    const int2 part = part_of(blocks, blockIdx.z, a.splits);
    const bool varies = tile.event < a.n_events && a.visible[tile.event] > 1;
    const Strided grad{a.grad, (long long)a.heads * a.dim, a.dim};
    load_seen(s_seen, a.mask, tile.begin, n_keys);
    __syncthreads();
    load_keys<T, DP>(s_k, a.k, piece_of<T>(a.k, a.dim), kv, tile.begin, a.dim, s_seen);
    load_keys<T, DP>(s_v, a.v, piece_of<T>(a.v, a.dim), kv, tile.begin, a.dim, s_seen);
    end_of_copies();
    const int piece_q = piece_of<T>(a.q, a.dim), piece_g = piece_of<T>(grad, a.dim);
    const auto load = [&](int step) {
        if (step < part.y * packs) {
            const int at = step % S, q0 = queries.x + step / packs * tokens, head0 = kv * a.group + step % packs * a.pack;
            const int n = min(tokens, queries.y - q0) * a.pack;
            load_queries<T, DP>(s_q + at * kRows * P, a.q, piece_q, head0, q0, n, a.pack, a.dim);
            load_queries<T, DP>(s_g + at * kRows * P, grad, piece_g, head0, q0, n, a.pack, a.dim);
            if (t < kRows) {
                float2 stat = t < n ? a.stats[(long long)(q0 + t / a.pack) * a.heads + head0 + t % a.pack] : make_float2(INFINITY, 0.f);
                stat.x += a.shift;
                s_stats_all[at][t] = stat;
            }
        }
        end_of_copies();
    };
    if (S > 1) load(part.x * packs);
    const float c = a.scale * kLog2e;
    float dk[DP / 8][4] = {}, dv[DP / 8][4] = {};
    const bool seen[2] = {s_seen[row0 + (lane_id() >> 2)] != 0, s_seen[row0 + (lane_id() >> 2) + 8] != 0};
    for (int step = part.x * packs; step < part.y * packs; step++) {
        __syncthreads();  // the buffers that are filled now have been read
        load(step + S - 1);
        copied<S - 1>();
        __syncthreads();
        const float *q_now = s_q + step % S * kRows * P + column0 * P, *g_now = s_g + step % S * kRows * P + column0 * P;
        const float2 *s_stats = s_stats_all[step % S] + column0 + 2 * (lane_id() & 3);
        float s[kBlocks][4], dp[kBlocks][4];
        dots<DP, kExact>(s, s_k + row0 * P, q_now, a.dim);
        dots<DP, kExact>(dp, s_v + row0 * P, g_now, a.dim);
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 stat = s_stats[8 * n + (i & 1)];  // infinity where there is no query
                s[n][i] = seen[i >> 1] ? mma::exp2_fast(fmaf(s[n][i], c, -stat.x)) : 0.f;
                dp[n][i] = seen[i >> 1] && varies ? s[n][i] * (dp[n][i] - stat.y) : 0.f;
            }
        weighted_rows<DP, kExact>(dv, s, g_now, a.dim);
        weighted_rows<DP, kExact>(dk, dp, q_now, a.dim);
    }
    copied<0>();
    __syncthreads();
    if (column0 > 0) {
        leave<DP>(s_q + row0 * P, dk);
        leave<DP>(s_g + row0 * P, dv);
    }
    __syncthreads();
    if (column0 > 0) return;
    const float one[2] = {1.f, 1.f};
    add<DP>(dk, s_q + row0 * P, one, one);
    add<DP>(dv, s_g + row0 * P, one, one);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = row0 + (lane_id() >> 2) + 8 * i;
        if (r >= n_keys) continue;
        if (!seen[i]) {  // a weight of zero does not make up for a query of NaN
#pragma unroll
            for (int n = 0; n < DP / 8; n++) dk[n][2 * i] = dk[n][2 * i + 1] = dv[n][2 * i] = dv[n][2 * i + 1] = 0.f;
        }
        const long long row = (long long)(tile.begin + r) * a.kv_heads + kv;
        if (a.splits > 1) {
            const long long at = ((long long)blockIdx.z * a.n_k * a.kv_heads + row) * a.dim;
            store_row<DP>(a.part + at, dk, i, a.scale, a.dim);
            store_row<DP>(a.part2 + at, dv, i, 1.f, a.dim);
        } else {
            store_row<DP>(static_cast<T *>(a.to) + row * a.dim, dk, i, a.scale, a.dim);
            store_row<DP>(static_cast<T *>(a.to2) + row * a.dim, dv, i, 1.f, a.dim);
        }
    }
}

// Sums the parts of one or two gradients, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
join_gradient_kernel(const float *__restrict__ part, const float *__restrict__ part2, T *__restrict__ to, T *__restrict__ to2,
                     long long n, int splits)
{
    pdl_begin();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float a = 0.f, b = 0.f;
    for (int s = 0; s < splits; s++) {
        a += part[s * n + i];
        if (part2 != nullptr) b += part2[s * n + i];
    }
    to[i] = from_float<T>(a);
    if (part2 != nullptr) to2[i] = from_float<T>(b);
}

// -------------------------------------------------------------------------------------------------------------- host
template <typename K>
int launch(K kernel, dim3 grid, size_t smem, cudaStream_t stream, const Args &a)
{
    HGC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    HGC_CUDA_TRY(launch_pdl(kernel, grid, kThreads, smem, stream, a));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

// How many parts the long axis is split into: as many as it takes to give every multiprocessor `per_sm` blocks, but parts of at
// least `least` steps of a mean event.  Depends on sizes alone, so that the workspace can be asked for.
int split_count(long long blocks, long long mean_steps, int per_sm, int least)
{
    const long long want = (long long)per_sm * sm_count() / (blocks > 0 ? blocks : 1);
    long long s = mean_steps / least;
    if (s > want) s = want;
    return s < 1 ? 1 : s > kMaxParts ? kMaxParts : (int)s;
}

// What a call of these sizes needs; the kernels and the workspace queries go by the same numbers.
struct Plan {
    int group, pack, splits, splits_mma, parts_mma, alternate, pack_few, rows_few, splits_few, splits_q, splits_q_mma, splits_k, splits_k_mma;
    long long tiles_q, tiles_k;
    bool close, close_q, close_k;
};

bool sizes_ok(int n_q, int n_k, int n_rs, int heads, int kv_heads, int dim)
{
    return n_q >= 0 && n_k >= 0 && n_rs >= 1 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && dim >= 1;
}
bool sizes_supported(int n_q, int n_k, int n_rs, int heads, int dim)
{
    return n_q <= kMaxCount && n_k <= kMaxCount && n_rs <= kMaxCount / 2 && heads <= 65535 && dim <= kMaxDim;
}

Plan plan_of(int n_q, int n_k, int n_rs, int heads, int kv_heads, int dim)
{
    Plan p;
    const int events = n_rs - 1;
    p.group = heads / kv_heads;
    p.pack = p.group <= kMaxPack ? p.group : 1;
    const int tokens = kRows / p.pack;
    p.tiles_q = tile_count(n_q, tokens, events);
    p.tiles_k = tile_count(n_k, kRows, events);
    const int some = events > 0 ? events : 1;
    // tiles that have rows, if the events are alike
    const auto filled = [&](int n, int rows) { return (long long)some * ((n / some + rows) / rows); };
    const long long steps_k = n_k / some / kRows, steps_q = n_q / some / tokens;
    // two blocks are resident: parts for many rounds of them, so that the last round counts little (a training step of three small events
    // with 4 and 6 blocks a multiprocessor 2836 us, with 8 and 20 2739)
    p.splits = split_count(filled(n_q, tokens) * (heads / p.pack), steps_k, 8, 4);
    const int mma_tokens = kMmaRows / p.pack;
    // events of no more rows than half a tile, and keys for both of its halves
    const long long steps_mma = n_k / some / mma_keys(dim);
    p.alternate = (long long)n_q <= (long long)some * mma_tokens && steps_mma >= 12;
    p.splits_mma = split_count(filled(n_q, p.alternate ? mma_tokens : 2 * mma_tokens) * (heads / p.pack), steps_mma, 6, 4);
    if (p.alternate && p.splits_mma > kMaxParts / 2) p.splits_mma = kMaxParts / 2;
    p.parts_mma = p.splits_mma * (p.alternate ? 2 : 1);
    // Where 16-bit types are better off with the products of this file: weights and their gradients are not rounded to 16 bits there.
    // In short calls, whose time is that of their launches, it costs nothing (32 events of 30 queries on 30 keys, forward and backward:
    // 28 and 70 us here, 32 and 68 there).  Of a few keys, gradients are differences of products that are much larger: off by 1.5 to 1.6
    // times their own rounding there, 1.2 here (8 events of 8192 queries on 8 keys of 8, 64 and 128 columns: 146, 427 and 805 us here,
    // 144, 199 and 263 there).  So is the gradient of narrow queries, whose keys have a large part in common, on any number
    // of keys: 1.5 to 1.6 for 8 and 16 columns.
    const long long mean_k = n_k / some, mean_q = n_q / some;
    p.close = mean_k <= kRows && mean_q * p.pack <= kRows && filled(n_q, tokens) * (heads / p.pack) <= 2 * sm_count();
    p.close_k = p.close || mean_k <= 16;
    p.close_q = p.close_k || dim <= 16;
    // where the queries of a mean event fit a block that holds them in registers
    p.pack_few = few_pack(p.group);
    p.rows_few = few_rows(n_q, events, p.pack_few);
    p.splits_few = p.rows_few > 0 ? split_count(filled(n_q, p.rows_few / p.pack_few) * (heads / p.pack_few), n_k / some / kFewStep, 20, 4) : 1;
    p.splits_q = split_count(filled(n_q, tokens) * (heads / p.pack), steps_k, 20, 4);
    p.splits_q_mma = split_count(filled(n_q, mma_tokens) * (heads / p.pack), n_k / some / kMmaGradStep, 4, 4);
    p.splits_k = split_count(filled(n_k, kRows) * kv_heads, steps_q, 20, 4);
    p.splits_k_mma = split_count(filled(n_k, kMmaRows) * kv_heads, n_q / some / (kMmaGradStep / p.pack), 2, 4);
    return p;
}

struct ForwardBuffers {
    int *counter = nullptr;
    float *part = nullptr, *part_lse = nullptr;
};
template <typename C> ForwardBuffers carve_forward(C &c, const Plan &p, int n_q, int heads, int dim)
{
    ForwardBuffers b;
    if constexpr (std::is_same_v<C, Carver>) b.counter = c.template take<int>(1);
    else c.template take<int>(1);
    int splits = p.splits > p.parts_mma ? p.splits : p.parts_mma;
    if (p.splits_few > splits) splits = p.splits_few;
    if (splits > 1) {
        const size_t rows = (size_t)splits * n_q * heads;
        if constexpr (std::is_same_v<C, Carver>) {
            b.part = c.template take<float>(rows * dim);
            b.part_lse = c.template take<float>(rows);
        } else {
            c.template take<float>(rows * dim);
            c.template take<float>(rows);
        }
    }
    return b;
}

struct BackwardBuffers {
    float2 *stats = nullptr;
    float *norms = nullptr, *bounds = nullptr, *part_q = nullptr, *part_k = nullptr, *part_v = nullptr;
    int *visible = nullptr;
};
template <typename C> BackwardBuffers carve_backward(C &c, const Plan &p, int n_q, int n_k, int n_rs, int heads, int kv_heads, int dim, int dtype)
{
    BackwardBuffers b;
    const int splits_q = p.splits_q > p.splits_q_mma ? p.splits_q : p.splits_q_mma, splits_k = p.splits_k > p.splits_k_mma ? p.splits_k : p.splits_k_mma;
    const size_t norms = dtype == HGC_FLOAT16 ? (size_t)n_q * heads : 0;
    const size_t rows = (size_t)n_q * heads, parts_q = splits_q > 1 ? splits_q * rows * dim : 0,
                 parts_k = splits_k > 1 ? (size_t)splits_k * n_k * kv_heads * dim : 0;
    if constexpr (std::is_same_v<C, Carver>) {
        b.stats = c.template take<float2>(rows);
        b.visible = c.template take<int>(n_rs);
        b.norms = c.template take<float>(norms);
        b.bounds = c.template take<float>(2 * (size_t)n_rs);
        b.part_q = c.template take<float>(parts_q);
        b.part_k = c.template take<float>(parts_k);
        b.part_v = c.template take<float>(parts_k);
    } else {
        c.template take<float2>(rows);
        c.template take<int>(n_rs);
        c.template take<float>(norms);
        c.template take<float>(2 * (size_t)n_rs);
        c.template take<float>(parts_q);
        c.template take<float>(parts_k);
        c.template take<float>(parts_k);
    }
    return b;
}

template <typename T, int DP> int run_forward(const Args &a, const Plan &p, cudaStream_t stream)
{
    const size_t smem = sizeof(float) * (1 + 2 * kStages<DP>) * kRows * kPitch<DP>;
    return launch(forward_kernel<T, DP>, dim3((unsigned)p.tiles_q, a.heads / a.pack, a.splits), smem, stream, a);
}

template <typename T> int join_gradient(const Args &a, long long n, cudaStream_t stream)
{
    if (a.splits == 1 || n == 0) return HGC_OK;
    HGC_CUDA_TRY(launch_pdl(join_gradient_kernel<T>, div_up(n, 256), 256, 0, stream, a.part, a.part2, static_cast<T *>(a.to), static_cast<T *>(a.to2), n,
                            a.splits));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

template <typename T, int DP> int run_grad_queries(const Args &a, const Plan &p, cudaStream_t stream)
{
    const size_t smem = sizeof(float) * (2 + 2 * kStages<DP>) * kRows * kPitch<DP>;
    return launch(grad_queries_kernel<T, DP>, dim3((unsigned)p.tiles_q, a.heads / a.pack, a.splits), smem, stream, a);
}
template <typename T, int DP> int run_grad_keys(const Args &a, const Plan &p, cudaStream_t stream)
{
    const size_t smem = sizeof(float) * (2 + 2 * kStages<DP>) * kRows * kPitch<DP>;
    return launch(grad_keys_kernel<T, DP>, dim3((unsigned)p.tiles_k, a.kv_heads, a.splits), smem, stream, a);
}

template <typename T> int forward_of(Args a, const Plan &p, int dtype, cudaStream_t stream)
{
    const bool few = few_takes(a, p.rows_few, dtype), mma = !few && !p.close && mma_takes(a, dtype);
    if (few) a.pack = p.pack_few;
    a.splits = few ? p.splits_few : mma ? p.splits_mma : p.splits;
    a.alternate = mma ? p.alternate : 0;
    const int parts = mma ? p.parts_mma : a.splits;
    if (const int rc = few ? few_forward(a, p.rows_few, dtype, stream)
                     : mma ? mma_forward(a, dtype, stream)
                     : a.dim <= 32 ? run_forward<T, 32>(a, p, stream)
                     : a.dim <= 64 ? run_forward<T, 64>(a, p, stream) : run_forward<T, 128>(a, p, stream))
        return rc;
    if (parts == 1) return HGC_OK;
    const long long rows = (long long)a.n_q * a.heads;
    HGC_CUDA_TRY(launch_pdl(join_forward_kernel<T>, div_up(rows, 8), 256, 0, stream, a.part, a.part_lse, static_cast<T *>(a.to), static_cast<T *>(a.rest),
                            a.lse, rows, a.dim,
                            parts));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

template <typename T>
int backward_of(Args a, const Plan &p, const BackwardBuffers &b, void *dq, void *dk, void *dv, int dtype, cudaStream_t stream)
{
    const auto aligned = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
    const bool takes = mma_takes(a, dtype) && aligned(dq) && aligned(dk) && aligned(dv), mma_q = takes && !p.close_q, mma_k = takes && !p.close_k,
               bounded = (mma_q || mma_k) && dtype == HGC_FLOAT16;
    // whole 16-byte vectors of rows where they are that
    constexpr int V = 16 / sizeof(T);
    int lanes_log2 = -1;
    if (a.dim % V == 0 && aligned(a.out) && aligned(a.out_rest) && aligned(a.grad) && (!bounded || (aligned(a.v.p) && a.v.row % V == 0 && a.v.head % V == 0)))
        for (lanes_log2 = 0; (V << lanes_log2) < a.dim; lanes_log2++) {}
    const int rows_a_block = kThreads / (lanes_log2 >= 0 ? 1 << lanes_log2 : 32) * kRowsALane;
    const int n_count = a.n_events > 0 ? a.n_events : 1, n_rows = div_up((long long)a.n_q * a.heads, rows_a_block),
              n_values = bounded ? div_up((long long)a.n_k * a.kv_heads, rows_a_block) : 0;
    if (bounded) HGC_CUDA_TRY(cudaMemsetAsync(b.bounds, 0, 2 * sizeof(float) * (size_t)n_count, stream));
    HGC_CUDA_TRY(launch_pdl(prepare_backward_kernel<T>, n_count + n_rows + n_values, kThreads, 0, stream, a, b.stats, b.visible, b.norms,
                            bounded ? b.bounds : nullptr, bounded ? kHalfShift : 0.f, n_count, n_rows, lanes_log2));
    HGC_LAUNCH_CHECK();
    a.stats = b.stats; a.visible = b.visible; a.norms = b.norms; a.bounds = b.bounds; a.shift = bounded ? kHalfShift : 0.f;
    if (dq != nullptr && a.n_q > 0) {
        a.to = dq; a.to2 = nullptr; a.part = b.part_q; a.part2 = nullptr; a.splits = mma_q ? p.splits_q_mma : p.splits_q;
        if (const int rc = mma_q ? mma_grad_queries(a, dtype, stream)
                         : a.dim <= 32 ? run_grad_queries<T, 32>(a, p, stream)
                         : a.dim <= 64 ? run_grad_queries<T, 64>(a, p, stream) : run_grad_queries<T, 128>(a, p, stream))
            return rc;
        if (const int rc = join_gradient<T>(a, (long long)a.n_q * a.heads * a.dim, stream)) return rc;
    }
    if (dk != nullptr && a.n_k > 0) {
        a.to = dk; a.to2 = dv; a.part = b.part_k; a.part2 = b.part_v; a.splits = mma_k ? p.splits_k_mma : p.splits_k;
        if (const int rc = mma_k ? mma_grad_keys(a, dtype, stream)
                         : a.dim <= 32 ? run_grad_keys<T, 32>(a, p, stream)
                         : a.dim <= 64 ? run_grad_keys<T, 64>(a, p, stream) : run_grad_keys<T, 128>(a, p, stream))
            return rc;
        if (const int rc = join_gradient<T>(a, (long long)a.n_k * a.kv_heads * a.dim, stream)) return rc;
    }
    return HGC_OK;
}

Args args_of(const void *q, const void *k, const void *v, const int *rs_q, const int *rs_k, const unsigned char *mask, float *lse, int n_q, int n_k,
             int n_rs, int heads, int kv_heads, int dim, const long long *strides, float scale, const Plan &p, void *workspace)
{
    const long long dq = (long long)heads * dim, dk = (long long)kv_heads * dim;
    Args a = {};
    a.q = strides ? Strided{q, strides[0], strides[1]} : Strided{q, dq, dim};
    a.k = strides ? Strided{k, strides[2], strides[3]} : Strided{k, dk, dim};
    a.v = strides ? Strided{v, strides[4], strides[5]} : Strided{v, dk, dim};
    a.rs_q = rs_q; a.rs_k = rs_k; a.mask = mask; a.lse = lse;
    a.status = static_cast<unsigned *>(workspace);
    a.n_q = n_q; a.n_k = n_k; a.n_events = n_rs - 1;
    a.heads = heads; a.kv_heads = kv_heads; a.group = p.group; a.pack = p.pack; a.dim = dim; a.scale = scale;
    return a;
}

// A workspace that comes along is left with a status word all the same.
int nothing_to_do(void *workspace, size_t bytes, cudaStream_t stream)
{
    if (workspace != nullptr && bytes >= sizeof(unsigned)) HGC_CUDA_TRY(cudaMemsetAsync(workspace, 0, sizeof(unsigned), stream));
    return HGC_OK;
}

bool scale_ok(float scale) { return scale > 0.f && scale <= 3.4e38f; }
bool strides_ok(const long long *strides)
{
    if (strides)
        for (int i = 0; i < 6; i++)
            if (strides[i] < 0) return false;
    return true;
}

}  // namespace
}  // namespace attn
}  // namespace hgc

using namespace hgc;
using namespace hgc::attn;

extern "C" size_t hgc_cross_attention_workspace_bytes(int n_q, int n_k, int n_rs, int n_heads, int n_kv_heads, int dim, int dtype)
{
    (void)dtype;
    if (!sizes_ok(n_q, n_k, n_rs, n_heads, n_kv_heads, dim) || !sizes_supported(n_q, n_k, n_rs, n_heads, dim)) return 0;
    Sizer s;
    carve_forward(s, plan_of(n_q, n_k, n_rs, n_heads, n_kv_heads, dim), n_q, n_heads, dim);
    return s.used;
}

extern "C" int hgc_cross_attention(const void *d_q, const void *d_k, const void *d_v, const int *d_q_row_splits, const int *d_k_row_splits,
                                   const unsigned char *d_key_mask, void *d_out, void *d_out_rest, float *d_lse, int n_q, int n_k, int n_rs, int n_heads,
                                   int n_kv_heads, int dim, const long long *strides, float scale, int dtype, void *workspace,
                                   size_t workspace_bytes, hgc_stream_t stream_)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (!sizes_ok(n_q, n_k, n_rs, n_heads, n_kv_heads, dim) || !scale_ok(scale) || !strides_ok(strides) || dtype < 0 || dtype > HGC_BFLOAT16)
        return HGC_ERR_INVALID_ARGUMENT;
    if (!sizes_supported(n_q, n_k, n_rs, n_heads, dim)) return HGC_ERR_UNSUPPORTED;
    if (n_q == 0) return nothing_to_do(workspace, workspace_bytes, stream);
    if (!d_q || !d_out || !d_lse || !d_q_row_splits || !d_k_row_splits || (n_k > 0 && (!d_k || !d_v))) return HGC_ERR_INVALID_ARGUMENT;
    if (const int rc = check_workspace(workspace, workspace_bytes,
                                       hgc_cross_attention_workspace_bytes(n_q, n_k, n_rs, n_heads, n_kv_heads, dim, dtype)))
        return rc;
    const Plan p = plan_of(n_q, n_k, n_rs, n_heads, n_kv_heads, dim);
    Args a = args_of(d_q, d_k, d_v, d_q_row_splits, d_k_row_splits, d_key_mask, d_lse, n_q, n_k, n_rs, n_heads, n_kv_heads, dim, strides, scale, p,
                     workspace);
    Carver carver(workspace);
    const ForwardBuffers b = carve_forward(carver, p, n_q, n_heads, dim);
    a.to = d_out; a.rest = dtype == HGC_FLOAT32 ? nullptr : d_out_rest; a.part = b.part; a.part_lse = b.part_lse; a.counter = b.counter;
    return dtype == HGC_FLOAT32 ? forward_of<float>(a, p, dtype, stream)
         : dtype == HGC_FLOAT16 ? forward_of<__half>(a, p, dtype, stream) : forward_of<__nv_bfloat16>(a, p, dtype, stream);
}

extern "C" size_t hgc_cross_attention_grad_workspace_bytes(int n_q, int n_k, int n_rs, int n_heads, int n_kv_heads, int dim, int dtype)
{
    if (!sizes_ok(n_q, n_k, n_rs, n_heads, n_kv_heads, dim) || !sizes_supported(n_q, n_k, n_rs, n_heads, dim)) return 0;
    Sizer s;
    carve_backward(s, plan_of(n_q, n_k, n_rs, n_heads, n_kv_heads, dim), n_q, n_k, n_rs, n_heads, n_kv_heads, dim, dtype);
    return s.used;
}

extern "C" int hgc_cross_attention_grad(const void *d_grad_out, const void *d_q, const void *d_k, const void *d_v, const void *d_out,
                                        const void *d_out_rest, const float *d_lse, const int *d_q_row_splits, const int *d_k_row_splits,
                                        const unsigned char *d_key_mask, void *d_grad_q, void *d_grad_k, void *d_grad_v, int n_q, int n_k,
                                        int n_rs, int n_heads, int n_kv_heads, int dim, const long long *strides, float scale, int dtype,
                                        void *workspace, size_t workspace_bytes, hgc_stream_t stream_)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (!sizes_ok(n_q, n_k, n_rs, n_heads, n_kv_heads, dim) || !scale_ok(scale) || !strides_ok(strides) || dtype < 0 || dtype > HGC_BFLOAT16)
        return HGC_ERR_INVALID_ARGUMENT;
    if (!sizes_supported(n_q, n_k, n_rs, n_heads, dim)) return HGC_ERR_UNSUPPORTED;
    if (n_q == 0 && n_k == 0) return nothing_to_do(workspace, workspace_bytes, stream);
    if (!d_q_row_splits || !d_k_row_splits || (n_q > 0 && (!d_grad_out || !d_q || !d_out || !d_lse)) || (n_k > 0 && (!d_k || !d_v)) ||
        !d_grad_k != !d_grad_v)
        return HGC_ERR_INVALID_ARGUMENT;
    if (const int rc = check_workspace(workspace, workspace_bytes,
                                       hgc_cross_attention_grad_workspace_bytes(n_q, n_k, n_rs, n_heads, n_kv_heads, dim, dtype)))
        return rc;
    const Plan p = plan_of(n_q, n_k, n_rs, n_heads, n_kv_heads, dim);
    Args a = args_of(d_q, d_k, d_v, d_q_row_splits, d_k_row_splits, d_key_mask, const_cast<float *>(d_lse), n_q, n_k, n_rs, n_heads, n_kv_heads, dim,
                     strides, scale, p, workspace);
    Carver carver(workspace);
    const BackwardBuffers b = carve_backward(carver, p, n_q, n_k, n_rs, n_heads, n_kv_heads, dim, dtype);
    a.grad = d_grad_out; a.out = d_out; a.out_rest = dtype == HGC_FLOAT32 ? nullptr : d_out_rest;
    return dtype == HGC_FLOAT32 ? backward_of<float>(a, p, b, d_grad_q, d_grad_k, d_grad_v, dtype, stream)
         : dtype == HGC_FLOAT16 ? backward_of<__half>(a, p, b, d_grad_q, d_grad_k, d_grad_v, dtype, stream)
                                : backward_of<__nv_bfloat16>(a, p, b, d_grad_q, d_grad_k, d_grad_v, dtype, stream);
}
