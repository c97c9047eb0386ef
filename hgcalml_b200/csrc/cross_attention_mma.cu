// Attention between two ragged sets of rows on the tensor cores, for 16-bit types.
//
// A block has 128 rows of queries (tokens times the heads that share a key head) and takes them through the keys of their event.
// Six warps: four hold a row of scores per lane and do the softmax, one copies keys and values, one issues the products.
// Scores S = Q K^T, weights P (16 bits) and sums O = P V live in tensor memory, 256 columns, so that two blocks share a
// multiprocessor and one's softmax runs under the other's products.
#include <cuda.h>
#include <atomic>

#include "cross_attention.cuh"
#include "mma_device.cuh"

namespace hgc {
namespace attn {
namespace {

using namespace mma;

constexpr int kBlock = 192;  // warps 0 to 3: rows; 4: copies; 5: products
constexpr int kTile = 64 * 2;  // bytes of a row of a tile in shared memory

struct Maps {
    CUtensorMap q, k, v, grad;
};

// Which of the keys [k0, k0 + 32 W) of a step can be seen, W words; all lanes of a warp call this.
template <int W>
__device__ __forceinline__ bool seen_words(unsigned (&seen)[W], const unsigned char *__restrict__ mask, int k0, int n)
{
    bool all = n >= 32 * W;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int key = 32 * w + lane_id();
        const bool in = key < n && (mask == nullptr || __ldg(mask + k0 + key) != 0);
        seen[w] = __ballot_sync(0xffffffffu, in);
        all = all && seen[w] == 0xffffffffu;
    }
    return all;
}

// Zeros for the rows of a tile that are not seen: what they hold may be infinite, and would stay so times a weight of zero.
template <int W>
__device__ __forceinline__ void clear_unseen(unsigned tile, int chunks, const unsigned (&seen)[W])
{
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (seen[w] == 0xffffffffu || (seen[w] >> lane_id()) & 1u) continue;
        for (int c = 0; c < chunks; c++)
#pragma unroll
            for (int i = 0; i < 8; i++)  // lanes start at different 16 bytes of their rows, to meet different banks
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                             :: "r"(tile + c * 32 * W * kTile + (32 * w + lane_id()) * kTile + ((i + lane_id()) & 7) * 16), "r"(0) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------------------- forward
template <int CHUNKS> struct Forward {
    static constexpr int kKeys = CHUNKS == 1 ? 128 : 64;  // of a step
    static constexpr int kStages = 2, kBarriers = 1 + 4 * kStages + 4;
    static constexpr int kTileBytes = kKeys * kTile * CHUNKS;
    static constexpr int kQueryBytes = kMmaRows * kTile * CHUNKS;
    static constexpr int kSmem = kQueryBytes + 2 * kStages * kTileBytes;
    // columns of tensor memory
    static constexpr int kScores = 0, kWeights = kKeys, kOut = CHUNKS == 1 ? 192 : 128, kColumns = 256;
};

template <typename T, int CHUNKS>
__global__ void __launch_bounds__(kBlock, 2)
forward_mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps)
{
    pdl_begin();
    using F = Forward<CHUNKS>;
    constexpr int N = F::kKeys, W = N / 32;
    extern __shared__ __align__(1024) char s_raw[];
    __shared__ __align__(8) unsigned long long s_bar[F::kBarriers];
    __shared__ unsigned s_tmem;
    __shared__ int s_gave_up;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int tokens = kMmaRows / a.pack, head0 = blockIdx.y * a.pack, kv = head0 / a.group;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_splits(a, t, kBlock);
    const Tile tile = find_tile(a.rs_q, a.n_q, a.n_events, tokens, blockIdx.x);
    if (tile.begin >= tile.end) return;
    const int n_rows = (tile.end - tile.begin) * a.pack;
    const int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    const int2 part = part_of(max(0, (keys.y - keys.x + N - 1) / N), blockIdx.z, a.splits);
    const int steps = part.y - part.x, first = keys.x + part.x * N;

    const unsigned s_q = smem_address(s_raw), s_k = s_q + F::kQueryBytes, s_v = s_k + F::kStages * F::kTileBytes;
    const unsigned bar = smem_address(s_bar), q_full = bar, k_full = bar + 8, k_empty = k_full + 8 * F::kStages, v_full = k_empty + 8 * F::kStages,
                   v_empty = v_full + 8 * F::kStages, s_full = v_empty + 8 * F::kStages, p_full = s_full + 8, o_full = p_full + 8,
                   all_done = o_full + 8;
    if (steps > 0) {
        if (t == 0) {
            for (int i = 0; i < F::kBarriers; i++) barrier_init(bar + 8 * i, bar + 8 * i == p_full ? 4 : 1);
            barrier_init_done();
            s_gave_up = 0;
        }
        if (warp == 5) tmem_alloc(&s_tmem, F::kColumns);
        before_sync();
        __syncthreads();
        after_sync();
    }
    volatile int *gave_up = &s_gave_up;
    const unsigned tmem = steps > 0 ? s_tmem : 0;

    if (warp == 4) {
        if (lane == 0 && steps > 0) {
            arrive_expect(q_full, CHUNKS * kTile * a.pack * tokens);
            for (int c = 0; c < CHUNKS; c++) copy_box(s_q + c * kMmaRows * kTile, &maps.q, q_full, 64 * c, head0, tile.begin);
            int k_copies = 0, v_copies = 0;
            for (int j = 0; j < steps; j++) {
                const int stage = j % F::kStages;
                const unsigned again = (j / F::kStages & 1) ^ 1;
                if (j >= F::kStages && !wait(k_empty + 8 * stage, again, gave_up, a.status)) break;
                arrive_expect(k_full + 8 * stage, F::kTileBytes);
                for (int c = 0; c < CHUNKS; c++)
                    copy_box(s_k + stage * F::kTileBytes + c * N * kTile, &maps.k, k_full + 8 * stage, 64 * c, kv, first + j * N);
                k_copies++;
                if (j >= F::kStages && !wait(v_empty + 8 * stage, again, gave_up, a.status)) break;
                arrive_expect(v_full + 8 * stage, F::kTileBytes);
                for (int c = 0; c < CHUNKS; c++)
                    copy_box(s_v + stage * F::kTileBytes + c * N * kTile, &maps.v, v_full + 8 * stage, 64 * c, kv, first + j * N);
                v_copies++;
            }
            // no copy is under way when the block leaves
            drain(q_full, 0);
            for (int j = max(0, k_copies - F::kStages); j < k_copies; j++) drain(k_full + 8 * (j % F::kStages), j / F::kStages & 1);
            for (int j = max(0, v_copies - F::kStages); j < v_copies; j++) drain(v_full + 8 * (j % F::kStages), j / F::kStages & 1);
        }
        __syncwarp();
    } else if (warp == 5) {
        const int depth = (a.dim + 15) / 16;
        const unsigned shape_s = shape<T>(N, false), shape_o = shape<T>(16 * depth, true);
        // scores of step j
        const auto scores = [&](int j) {
            const int stage = j % F::kStages;
            const bool ok = wait_warp(k_full + 8 * stage, j / F::kStages & 1, gave_up, a.status);
            after_sync();
            if (lane == 0 && ok) {
                product_along(tmem + F::kScores, s_q, kMmaRows * kTile, s_k + stage * F::kTileBytes, N * kTile, depth, shape_s);
                arrive_when_done(s_full);
                arrive_when_done(k_empty + 8 * stage);
            }
        };
        if (steps > 0 && wait_warp(q_full, 0, gave_up, a.status)) {
            scores(0);
            for (int j = 0; j < steps; j++) {
                const int stage = j % F::kStages;
                unsigned seen[W];
                const bool all = seen_words<W>(seen, a.mask, first + j * N, keys.y - (first + j * N));
                if (!wait_warp(v_full + 8 * stage, j / F::kStages & 1, gave_up, a.status)) break;
                if (!all) {
                    clear_unseen<W>(s_v + stage * F::kTileBytes, CHUNKS, seen);
                    writes_before_products();
                    __syncwarp();
                }
                if (!wait_warp(p_full, j & 1, gave_up, a.status)) break;
                after_sync();
                if (j + 1 < steps) scores(j + 1);
                if (lane == 0 && !*gave_up) {
                    product_over(tmem + F::kOut, tmem + F::kWeights, s_v + stage * F::kTileBytes, N * kTile, N / 16, shape_o, j > 0);
                    arrive_when_done(o_full);
                    arrive_when_done(v_empty + 8 * stage);
                }
                __syncwarp();
            }
            if (lane == 0) {  // no product is under way when the tensor memory is freed
                arrive_when_done(all_done);
                drain(all_done, 0);
            }
            __syncwarp();
        }
    } else {
        const unsigned rows = tmem + ((unsigned)warp << 21);  // lane 32 w of tensor memory
        const bool idle = warp * 32 >= n_rows;                // none of the warp's rows counts
        const float c = a.scale * kLog2e;
        float top = -INFINITY, sum = 0.f;
        for (int j = 0; j < steps; j++) {
            unsigned seen[W];
            const bool all = seen_words<W>(seen, a.mask, first + j * N, keys.y - (first + j * N));
            if (!wait_warp(s_full, j & 1, gave_up, a.status)) break;
            after_sync();
            if (!idle) {
                unsigned s[W][32];
#pragma unroll
                for (int w = 0; w < W; w++) tmem_load32(s[w], rows + F::kScores + 32 * w);
                tmem_loaded();
#pragma unroll
                for (int w = 0; w < W; w++) use_after(s[w]);
                if (!all) {
#pragma unroll
                    for (int w = 0; w < W; w++)
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (!((seen[w] >> i) & 1u)) s[w][i] = 0xff800000u;
                }
                float m[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int i = 0; i < 32; i++) m[i & 3] = fmaxf(m[i & 3], __uint_as_float(s[w][i]));
                const float next = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                if (j > 0 && !wait_warp(o_full, (j - 1) & 1, gave_up, a.status)) break;
                // The sums are scaled again only where a row's maximum has grown by more than 2^8: weights up to that
                // lose nothing in either type.
                const bool grown = (next - top) * c > 8.f;
                if (j == 0) top = next;
                else if (__any_sync(0xffffffffu, grown)) {
                    after_sync();
                    const float shrink = exp2_fast((top - (next == -INFINITY ? 0.f : next)) * c);
                    top = next;
                    sum *= shrink;
                    for (int d = 0; d < a.dim; d += 16) {
                        unsigned o[16];
                        tmem_load16(o, rows + F::kOut + d);
                        tmem_loaded();
                        use_after(o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                        tmem_store16(rows + F::kOut + d, o);
                    }
                }
                const float base = (top == -INFINITY ? 0.f : top) * c;
                float part_sum[4] = {};
#pragma unroll
                for (int w = 0; w < W; w++) {
                    unsigned p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float x = exp2_fast(fmaf(__uint_as_float(s[w][2 * i]), c, -base)), y = exp2_fast(fmaf(__uint_as_float(s[w][2 * i + 1]), c, -base));
                        part_sum[i & 3] += x + y;
                        p[i] = pack2<T>(x, y);
                    }
                    tmem_store16(rows + F::kWeights + 16 * w, p);
                }
                sum += (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
                tmem_stored();
            } else if (j > 0 && !wait_warp(o_full, (j - 1) & 1, gave_up, a.status)) {
                break;
            }
            before_sync();
            __syncwarp();
            if (lane == 0) arrive(p_full);
        }
        const bool done = steps > 0 && wait_warp(o_full, (steps - 1) & 1, gave_up, a.status);
        if (done) after_sync();
        const int r = t;
        const bool store = r < n_rows;
        const long long row = (long long)(tile.begin + r / a.pack) * a.heads + head0 + r % a.pack;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const long long all_rows = (long long)a.n_q * a.heads;
        if (store) {
            float *lse = a.splits > 1 ? a.part_lse + blockIdx.z * all_rows : a.lse;
            lse[row] = sum == 0.f ? -INFINITY : top * a.scale + logf(sum);
        }
        if (!idle)
            for (int d = 0; d < a.dim; d += 16) {
                unsigned o[16];
                if (done) {
                    tmem_load16(o, rows + F::kOut + d);
                    tmem_loaded();
                    use_after(o);
                }
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = done ? __uint_as_float(o[i]) * inv : 0.f;
                if (store && a.splits > 1 && done) {  // a part without keys has no weight
                    float4 *to = reinterpret_cast<float4 *>(a.part + (blockIdx.z * all_rows + row) * a.dim + d);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (d + 4 * i < a.dim) to[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                } else if (store && a.splits == 1) {
                    uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(a.to) + row * a.dim + d);
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (d + 8 * i < a.dim)
                            to[i] = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]), pack2<T>(v[8 * i + 4], v[8 * i + 5]),
                                               pack2<T>(v[8 * i + 6], v[8 * i + 7]));
                }
                __syncwarp();
            }
    }
    if (steps > 0) {
        before_sync();
        __syncthreads();
        after_sync();
        if (warp == 5) tmem_free(tmem, F::kColumns);
    }
}

// ------------------------------------------------------------------------------------------------------------ backward
// Half precision reaches down to 2^-24 only, and a weight among many keys lies below that: weights are held 2^14 times as large
// there, and their gradients are scaled by a power of two under which none can overflow (|do.v - delta| <= 2 max|do| max|v|).
// Both factors are taken out of the float32 sums.
template <typename T> struct Range { static constexpr float kShift = 0.f; };
template <> struct Range<__half> { static constexpr float kShift = kHalfShift; };

template <typename T> __device__ __forceinline__ float slope_factor(const Args &a)
{
    if (Range<T>::kShift == 0.f) return 1.f;
    const float bound = sqrtf(__ldg(a.bounds)) * sqrtf(__ldg(a.bounds + 1));
    return bound > 0.f && bound < 1e30f ? exp2f(-ceilf(log2f(bound))) : 1.f;
}

// Rows [from, to) of a tile as zeros; a whole warp.
__device__ __forceinline__ void clear_rows(unsigned tile, int chunks, int tile_rows, int from, int to)
{
    for (int c = 0; c < chunks; c++)
        for (int i = from * 8 + lane_id(); i < to * 8; i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(tile + c * tile_rows * kTile + i * 16), "r"(0) : "memory");
}

// 16 columns of a row of a gradient
template <typename T>
__device__ __forceinline__ void store16(void *to, float *part, long long at, int d, int dim, const unsigned (&v)[16], float factor)
{
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = __uint_as_float(v[i]) * factor;
    if (part != nullptr) {
        float4 *p = reinterpret_cast<float4 *>(part + at + d);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (d + 4 * i < dim) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
        uint4 *p = reinterpret_cast<uint4 *>(static_cast<T *>(to) + at + d);
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (d + 8 * i < dim)
                p[i] = make_uint4(pack2<T>(x[8 * i], x[8 * i + 1]), pack2<T>(x[8 * i + 2], x[8 * i + 3]), pack2<T>(x[8 * i + 4], x[8 * i + 5]),
                                  pack2<T>(x[8 * i + 6], x[8 * i + 7]));
    }
}

// dq: as the forward pass, with S = Q K^T and dP = dO V^T, from which dS (16 bits) goes into dQ += dS K.  64 keys a step, so that two
// blocks fit a multiprocessor.  Wide heads: dS takes the place of S, and V has one stage.
template <int CHUNKS> struct GradQueries {
    static constexpr int kKeys = kMmaGradStep, kStagesK = 2, kStagesV = CHUNKS == 1 ? 2 : 1;
    static constexpr int kTileBytes = kKeys * kTile * CHUNKS, kQueryBytes = kMmaRows * kTile * CHUNKS;
    static constexpr int kTiles = 2 * kQueryBytes + (kStagesK + kStagesV) * kTileBytes, kSmem = kTiles + 256;
    static constexpr bool kInPlace = CHUNKS == 2;
    static constexpr int kScores = 0, kProducts = 64, kSlopes = kInPlace ? 0 : 128, kOut = kInPlace ? 128 : 160, kColumns = 256;
    static constexpr int kBarriers = 1 + 2 * kStagesK + 2 * kStagesV + 4;
};

template <typename T, int CHUNKS>
__global__ void __launch_bounds__(kBlock, 2)
grad_queries_mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps)
{
    pdl_begin();
    using F = GradQueries<CHUNKS>;
    constexpr int N = F::kKeys, W = N / 32;
    extern __shared__ __align__(1024) char s_raw[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int tokens = kMmaRows / a.pack, head0 = blockIdx.y * a.pack, kv = head0 / a.group;
    const Tile tile = find_tile(a.rs_q, a.n_q, a.n_events, tokens, blockIdx.x);
    if (tile.begin >= tile.end) return;
    const int n_rows = (tile.end - tile.begin) * a.pack;
    int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    if (tile.event < a.n_events && a.visible[tile.event] < 2) keys.y = keys.x;
    const int2 part = part_of(max(0, (keys.y - keys.x + N - 1) / N), blockIdx.z, a.splits);
    const int steps = part.y - part.x, first = keys.x + part.x * N;

    const unsigned s_q = smem_address(s_raw), s_g = s_q + F::kQueryBytes, s_k = s_g + F::kQueryBytes, s_v = s_k + F::kStagesK * F::kTileBytes;
    const unsigned bar = s_q + F::kTiles, q_full = bar, k_full = bar + 8, k_empty = k_full + 8 * F::kStagesK, v_full = k_empty + 8 * F::kStagesK,
                   v_empty = v_full + 8 * F::kStagesV, s_full = v_empty + 8 * F::kStagesV, p_full = s_full + 8, o_full = p_full + 8, all_done = o_full + 8;
    static_assert(8 * F::kBarriers + 8 <= 256, "room behind the tiles");
    unsigned *s_tmem = reinterpret_cast<unsigned *>(s_raw + F::kTiles + 8 * F::kBarriers);
    volatile int *gave_up = reinterpret_cast<volatile int *>(s_tmem + 1);
    if (steps > 0) {
        if (t == 0) {
            for (int i = 0; i < F::kBarriers; i++) barrier_init(bar + 8 * i, bar + 8 * i == p_full ? 4 : 1);
            barrier_init_done();
            *gave_up = 0;
        }
        if (warp == 5) tmem_alloc(s_tmem, F::kColumns);
        before_sync();
        __syncthreads();
        after_sync();
    }
    const unsigned tmem = steps > 0 ? *s_tmem : 0;

    if (warp == 4) {
        if (lane == 0 && steps > 0) {
            arrive_expect(q_full, 2 * CHUNKS * kTile * a.pack * tokens);
            for (int c = 0; c < CHUNKS; c++) {
                copy_box(s_q + c * kMmaRows * kTile, &maps.q, q_full, 64 * c, head0, tile.begin);
                copy_box(s_g + c * kMmaRows * kTile, &maps.grad, q_full, 64 * c, head0, tile.begin);
            }
            int k_copies = 0, v_copies = 0;
            for (int j = 0; j < steps; j++) {
                const int sk = j % F::kStagesK, sv = j % F::kStagesV;
                if (j >= F::kStagesK && !wait(k_empty + 8 * sk, (j / F::kStagesK & 1) ^ 1, gave_up, a.status)) break;
                arrive_expect(k_full + 8 * sk, F::kTileBytes);
                for (int c = 0; c < CHUNKS; c++) copy_box(s_k + sk * F::kTileBytes + c * N * kTile, &maps.k, k_full + 8 * sk, 64 * c, kv, first + j * N);
                k_copies++;
                if (j >= F::kStagesV && !wait(v_empty + 8 * sv, (j / F::kStagesV & 1) ^ 1, gave_up, a.status)) break;
                arrive_expect(v_full + 8 * sv, F::kTileBytes);
                for (int c = 0; c < CHUNKS; c++) copy_box(s_v + sv * F::kTileBytes + c * N * kTile, &maps.v, v_full + 8 * sv, 64 * c, kv, first + j * N);
                v_copies++;
            }
            drain(q_full, 0);
            for (int j = max(0, k_copies - F::kStagesK); j < k_copies; j++) drain(k_full + 8 * (j % F::kStagesK), j / F::kStagesK & 1);
            for (int j = max(0, v_copies - F::kStagesV); j < v_copies; j++) drain(v_full + 8 * (j % F::kStagesV), j / F::kStagesV & 1);
        }
        __syncwarp();
    } else if (warp == 5) {
        const int depth = (a.dim + 15) / 16;
        const unsigned shape_s = shape<T>(N, false), shape_o = shape<T>(16 * depth, true);
        const auto scores = [&](int j) {
            const int sk = j % F::kStagesK, sv = j % F::kStagesV;
            unsigned seen[W];
            const bool all = seen_words<W>(seen, a.mask, first + j * N, keys.y - (first + j * N));
            bool ok = wait_warp(k_full + 8 * sk, j / F::kStagesK & 1, gave_up, a.status);
            if (ok && !all) {
                clear_unseen<W>(s_k + sk * F::kTileBytes, CHUNKS, seen);
                writes_before_products();
                __syncwarp();
            }
            ok = ok && wait_warp(v_full + 8 * sv, j / F::kStagesV & 1, gave_up, a.status);
            after_sync();
            if (lane == 0 && ok) {
                product_along(tmem + F::kScores, s_q, kMmaRows * kTile, s_k + sk * F::kTileBytes, N * kTile, depth, shape_s);
                product_along(tmem + F::kProducts, s_g, kMmaRows * kTile, s_v + sv * F::kTileBytes, N * kTile, depth, shape_s);
                arrive_when_done(s_full);
                arrive_when_done(v_empty + 8 * sv);
            }
            __syncwarp();
        };
        if (steps > 0 && wait_warp(q_full, 0, gave_up, a.status)) {
            scores(0);
            for (int j = 0; j < steps; j++) {
                const int sk = j % F::kStagesK;
                if (!wait_warp(p_full, j & 1, gave_up, a.status)) break;
                after_sync();
                if (!F::kInPlace && j + 1 < steps) scores(j + 1);
                if (lane == 0 && !*gave_up) {
                    product_over(tmem + F::kOut, tmem + F::kSlopes, s_k + sk * F::kTileBytes, N * kTile, N / 16, shape_o, j > 0);
                    arrive_when_done(o_full);
                    arrive_when_done(k_empty + 8 * sk);
                }
                __syncwarp();
                if (F::kInPlace && j + 1 < steps) {
                    if (!wait_warp(o_full, j & 1, gave_up, a.status)) break;
                    scores(j + 1);
                }
            }
            if (lane == 0) {
                arrive_when_done(all_done);
                drain(all_done, 0);
            }
            __syncwarp();
        }
    } else {
        const unsigned rows = tmem + ((unsigned)warp << 21);
        const bool idle = warp * 32 >= n_rows, store = t < n_rows;
        const long long row = (long long)(tile.begin + t / a.pack) * a.heads + head0 + t % a.pack;
        const float c = a.scale * kLog2e, factor = slope_factor<T>(a);
        const float2 stat = store ? a.stats[row] : make_float2(INFINITY, 0.f);
        const float shift = stat.x, delta = stat.y * factor;
        for (int j = 0; j < steps; j++) {
            unsigned seen[W];
            const bool all = seen_words<W>(seen, a.mask, first + j * N, keys.y - (first + j * N));
            if (!wait_warp(s_full, j & 1, gave_up, a.status)) break;
            after_sync();
            unsigned slopes[W][16];
            if (!idle) {
#pragma unroll
                for (int w = 0; w < W; w++) {
                    unsigned s[32], g[32];
                    tmem_load32(s, rows + F::kScores + 32 * w);
                    tmem_load32(g, rows + F::kProducts + 32 * w);
                    tmem_loaded();
                    use_after(s);
                    use_after(g);
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const float p = exp2_fast(fmaf(__uint_as_float(s[i]), c, -shift));
                        const float d = Range<T>::kShift == 0.f ? __uint_as_float(g[i]) - delta : fmaf(__uint_as_float(g[i]), factor, -delta);
                        s[i] = __float_as_uint(p * d);
                    }
                    if (!all) {
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (!((seen[w] >> i) & 1u)) s[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) slopes[w][i] = pack2<T>(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
                }
            }
            // where the slopes go, the last step's product has been
            if (!F::kInPlace && j > 0 && !wait_warp(o_full, (j - 1) & 1, gave_up, a.status)) break;
            if (!idle) {
                after_sync();
#pragma unroll
                for (int w = 0; w < W; w++) tmem_store16(rows + F::kSlopes + 16 * w, slopes[w]);
                tmem_stored();
            }
            before_sync();
            __syncwarp();
            if (lane == 0) arrive(p_full);
        }
        const bool done = steps > 0 && wait_warp(o_full, (steps - 1) & 1, gave_up, a.status);
        if (done) after_sync();
        const float back = a.scale * exp2f(-Range<T>::kShift) / factor;
        float *to_part = a.splits > 1 ? a.part + blockIdx.z * (long long)a.n_q * a.heads * a.dim : nullptr;
        if (!idle)
            for (int d = 0; d < a.dim; d += 16) {
                unsigned o[16] = {};
                if (done) {
                    tmem_load16(o, rows + F::kOut + d);
                    tmem_loaded();
                    use_after(o);
                }
                if (store) store16<T>(a.to, to_part, row * a.dim, d, a.dim, o, back);
                __syncwarp();
            }
    }
    if (steps > 0) {
        before_sync();
        __syncthreads();
        after_sync();
        if (warp == 5) tmem_free(tmem, F::kColumns);
    }
}

// dk and dv of 128 keys: a lane has a key, columns are queries.  S^T = K Q^T and dP^T = V dO^T give P^T and dS^T (16 bits, in their
// places), which go into dV += P^T dO and dK += dS^T Q straight from tensor memory.  Narrow heads: 256 columns and two blocks on a
// multiprocessor.  Wide ones: all 512 columns, and two groups of four warps that take the steps in turn.
template <int CHUNKS> struct GradKeys {
    static constexpr int kQueries = kMmaGradStep, kGroups = CHUNKS, kStages = CHUNKS == 1 ? 2 : 3, kThreads = 128 * kGroups + 64;
    static constexpr int kTileBytes = kQueries * kTile * CHUNKS, kKeyBytes = kMmaRows * kTile * CHUNKS;
    static constexpr int kTiles = 2 * kKeyBytes + 2 * kStages * kTileBytes, kStats = kGroups * kQueries * 8, kSmem = kTiles + kStats + 256;
    static constexpr int kDk = 128 * kGroups, kDv = kDk + 64 * CHUNKS, kColumns = 256 * CHUNKS;
    static constexpr int kBarriers = 1 + 2 * kStages + 3 * kGroups + 1;
};

template <typename T, int CHUNKS>
__global__ void __launch_bounds__(GradKeys<CHUNKS>::kThreads, CHUNKS == 1 ? 2 : 1)
grad_keys_mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps)
{
    pdl_begin();
    using F = GradKeys<CHUNKS>;
    constexpr int N = F::kQueries, G = F::kGroups;
    extern __shared__ __align__(1024) char s_raw[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, kv = blockIdx.y;
    const Tile tile = find_tile(a.rs_k, a.n_k, a.n_events, kMmaRows, blockIdx.x);
    if (tile.begin >= tile.end) return;
    const int n_keys = tile.end - tile.begin, tokens = N / a.pack, packs = a.group / a.pack;
    const int2 queries = rows_of(a.rs_q, a.n_q, a.n_events, tile.event);
    const int2 part = part_of(max(0, (queries.y - queries.x + tokens - 1) / tokens), blockIdx.z, a.splits);
    const int begin = part.x * packs, steps = part.y * packs - begin;
    const bool varies = tile.event < a.n_events && a.visible[tile.event] > 1;

    const unsigned s_k = smem_address(s_raw), s_v = s_k + F::kKeyBytes, s_q = s_v + F::kKeyBytes, s_g = s_q + F::kStages * F::kTileBytes;
    const unsigned bar = s_k + F::kTiles + F::kStats, k_full = bar, q_full = bar + 8, q_empty = q_full + 8 * F::kStages, s_full = q_empty + 8 * F::kStages,
                   p_full = s_full + 8 * G, used = p_full + 8 * G, all_done = used + 8 * G;
    static_assert(8 * F::kBarriers + 8 <= 256, "room behind the tiles");
    float2 *s_stats = reinterpret_cast<float2 *>(s_raw + F::kTiles);
    unsigned *s_tmem = reinterpret_cast<unsigned *>(s_raw + F::kTiles + F::kStats + 8 * F::kBarriers);
    volatile int *gave_up = reinterpret_cast<volatile int *>(s_tmem + 1);
    if (steps > 0) {
        if (t == 0) {
            for (int i = 0; i < F::kBarriers; i++) {
                const unsigned b = bar + 8 * i;
                barrier_init(b, b >= p_full && b < used ? 4 : 1);
            }
            barrier_init_done();
            *gave_up = 0;
        }
        if (warp == 4 * G + 1) tmem_alloc(s_tmem, F::kColumns);
        before_sync();
        __syncthreads();
        after_sync();
    }
    const unsigned tmem = steps > 0 ? *s_tmem : 0;

    if (warp == 4 * G) {
        if (lane == 0 && steps > 0) {
            arrive_expect(k_full, 2 * F::kKeyBytes);
            for (int c = 0; c < CHUNKS; c++) {
                copy_box(s_k + c * kMmaRows * kTile, &maps.k, k_full, 64 * c, kv, tile.begin);
                copy_box(s_v + c * kMmaRows * kTile, &maps.v, k_full, 64 * c, kv, tile.begin);
            }
            int copies = 0;
            for (int j = 0; j < steps; j++) {
                const int stage = j % F::kStages, step = begin + j;
                if (j >= F::kStages && !wait(q_empty + 8 * stage, (j / F::kStages & 1) ^ 1, gave_up, a.status)) break;
                arrive_expect(q_full + 8 * stage, 2 * CHUNKS * kTile * a.pack * tokens);
                const int q0 = queries.x + step / packs * tokens, head0 = kv * a.group + step % packs * a.pack;
                for (int c = 0; c < CHUNKS; c++) {
                    copy_box(s_q + stage * F::kTileBytes + c * N * kTile, &maps.q, q_full + 8 * stage, 64 * c, head0, q0);
                    copy_box(s_g + stage * F::kTileBytes + c * N * kTile, &maps.grad, q_full + 8 * stage, 64 * c, head0, q0);
                }
                copies++;
            }
            drain(k_full, 0);
            for (int j = max(0, copies - F::kStages); j < copies; j++) drain(q_full + 8 * (j % F::kStages), j / F::kStages & 1);
        }
        __syncwarp();
    } else if (warp == 4 * G + 1) {
        const int depth = (a.dim + 15) / 16;
        const unsigned shape_s = shape<T>(N, false), shape_o = shape<T>(16 * depth, true);
        const auto scores = [&](int j) {
            const int stage = j % F::kStages, g = j % G;
            const bool ok = wait_warp(q_full + 8 * stage, j / F::kStages & 1, gave_up, a.status);
            // rows of another event are not summed over, whatever they hold
            const int n = min(tokens, queries.y - (queries.x + (begin + j) / packs * tokens)) * a.pack;
            if (ok && n < a.pack * tokens) {
                clear_rows(s_q + stage * F::kTileBytes, CHUNKS, N, n, a.pack * tokens);
                clear_rows(s_g + stage * F::kTileBytes, CHUNKS, N, n, a.pack * tokens);
                writes_before_products();
                __syncwarp();
            }
            after_sync();
            if (lane == 0 && ok) {
                product_along(tmem + 128 * g, s_k, kMmaRows * kTile, s_q + stage * F::kTileBytes, N * kTile, depth, shape_s);
                product_along(tmem + 128 * g + 64, s_v, kMmaRows * kTile, s_g + stage * F::kTileBytes, N * kTile, depth, shape_s);
                arrive_when_done(s_full + 8 * g);
            }
            __syncwarp();
        };
        if (steps > 0) {
            if (a.pack * tokens < N) {  // rows that no copy writes
                for (int i = 0; i < F::kStages; i++) {
                    clear_rows(s_q + i * F::kTileBytes, CHUNKS, N, a.pack * tokens, N);
                    clear_rows(s_g + i * F::kTileBytes, CHUNKS, N, a.pack * tokens, N);
                }
                writes_before_products();
                __syncwarp();
            }
            if (wait_warp(k_full, 0, gave_up, a.status)) {
                for (int j = 0; j < min(G, steps); j++) scores(j);
                for (int j = 0; j < steps; j++) {
                    const int stage = j % F::kStages, g = j % G;
                    if (!wait_warp(p_full + 8 * g, j / G & 1, gave_up, a.status)) break;
                    after_sync();
                    if (lane == 0 && !*gave_up) {
                        product_over(tmem + F::kDv, tmem + 128 * g, s_g + stage * F::kTileBytes, N * kTile, N / 16, shape_o, j > 0);
                        product_over(tmem + F::kDk, tmem + 128 * g + 64, s_q + stage * F::kTileBytes, N * kTile, N / 16, shape_o, j > 0);
                        arrive_when_done(used + 8 * g);
                        arrive_when_done(q_empty + 8 * stage);
                    }
                    __syncwarp();
                    if (j + G < steps) {
                        if (!wait_warp(used + 8 * g, j / G & 1, gave_up, a.status)) break;
                        scores(j + G);
                    }
                }
                if (lane == 0) {
                    arrive_when_done(all_done);
                    drain(all_done, 0);
                }
                __syncwarp();
            }
        }
    } else {
        const int g = warp >> 2, r = t & 127;
        const unsigned lanes = tmem + ((unsigned)(warp & 3) << 21), rows = lanes + 128 * g;
        const bool store = r < n_keys;
        const unsigned seen = store && (a.mask == nullptr || __ldg(a.mask + tile.begin + r) != 0) ? 0xffffffffu : 0u;
        const float c = a.scale * kLog2e, factor = slope_factor<T>(a);
        float2 *stats = s_stats + g * N;
        for (int j = g; j < steps; j += G) {
            const int step = begin + j, q0 = queries.x + step / packs * tokens, head0 = kv * a.group + step % packs * a.pack;
            float2 mine = make_float2(INFINITY, 0.f);
            if (r < min(tokens, queries.y - q0) * a.pack) {
                mine = a.stats[(long long)(q0 + r / a.pack) * a.heads + head0 + r % a.pack];
                mine.y *= factor;
            }
            asm volatile("bar.sync %0, 128;" :: "r"(1 + g) : "memory");  // the last step's have been read
            if (r < N) stats[r] = mine;
            asm volatile("bar.sync %0, 128;" :: "r"(1 + g) : "memory");
            if (wait_warp(s_full + 8 * g, j / G & 1, gave_up, a.status)) {  // else on to the next step: the group's barriers count on all warps
                after_sync();
#pragma unroll
                for (int w = 0; w < N / 32; w++) {
                    unsigned s[32], d[32], p[16], q[16];
                    tmem_load32(s, rows + 32 * w);
                    tmem_load32(d, rows + 64 + 32 * w);
                    tmem_loaded();
                    use_after(s);
                    use_after(d);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float4 st = *reinterpret_cast<const float4 *>(stats + 32 * w + i);
                        const float p0 = exp2_fast(fmaf(__uint_as_float(s[i]), c, -st.x)), p1 = exp2_fast(fmaf(__uint_as_float(s[i + 1]), c, -st.z));
                        float d0 = __uint_as_float(d[i]), d1 = __uint_as_float(d[i + 1]);
                        d0 = Range<T>::kShift == 0.f ? d0 - st.y : fmaf(d0, factor, -st.y);
                        d1 = Range<T>::kShift == 0.f ? d1 - st.w : fmaf(d1, factor, -st.w);
                        p[i / 2] = pack2<T>(p0, p1) & seen;
                        q[i / 2] = pack2<T>(p0 * d0, p1 * d1) & seen;
                    }
                    // in place: these columns have been read, by the lanes that own their rows
                    tmem_store16(rows + 16 * w, p);
                    tmem_store16(rows + 64 + 16 * w, q);
                }
                tmem_stored();
            }
            before_sync();
            __syncwarp();
            if (lane == 0) arrive(p_full + 8 * g);
        }
        // the sums are complete when the last step's products are: that of this group's own last step waits for it
        bool done = steps > 0;
        if (steps > 0) done = wait_warp(all_done, 0, gave_up, a.status);
        if (done) after_sync();
        const long long at = ((long long)(tile.begin + r) * a.kv_heads + kv) * a.dim, all = (long long)a.n_k * a.kv_heads * a.dim;
        const float back = exp2f(-Range<T>::kShift);
        // one group writes dv, the last one dk
        for (int which = 0; which < 2; which++) {
            if (G == 2 && which != g) continue;
            float *to_part = a.splits > 1 ? (which == 0 ? a.part2 : a.part) + blockIdx.z * all : nullptr;
            const float f = which == 0 ? back : varies ? a.scale * back / factor : 0.f;
            for (int d = 0; d < a.dim; d += 16) {
                unsigned o[16] = {};
                if (done && (which == 0 || varies)) {
                    tmem_load16(o, lanes + (which == 0 ? F::kDv : F::kDk) + d);
                    tmem_loaded();
                    use_after(o);
                }
                if (store) store16<T>(which == 0 ? a.to2 : a.to, to_part, at, d, a.dim, o, f);
                __syncwarp();
            }
        }
    }
    if (steps > 0) {
        before_sync();
        __syncthreads();
        after_sync();
        if (warp == 4 * G + 1) tmem_free(tmem, F::kColumns);
    }
}

// -------------------------------------------------------------------------------------------------------------- host
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled()
{
    static std::atomic<void *> entry{nullptr};
    void *p = entry.load(std::memory_order_acquire);
    if (p == nullptr) {
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            return nullptr;
        entry.store(p, std::memory_order_release);
    }
    return reinterpret_cast<EncodeTiled>(p);
}

// Boxes of 64 columns x `heads` heads x `rows` rows of a tensor of n rows.
int map_of(CUtensorMap *map, const Strided &s, int dtype, int dim, int n_heads, int n, int heads, int rows)
{
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) {
        set_cuda_error(cudaErrorNotSupported);
        return HGC_ERR_CUDA;
    }
    const cuuint64_t size[3] = {(cuuint64_t)dim, (cuuint64_t)n_heads, (cuuint64_t)n};
    const cuuint64_t stride[2] = {(cuuint64_t)s.head * 2, (cuuint64_t)s.row * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)rows}, step[3] = {1, 1, 1};
    const CUresult rc = encode(map, dtype == HGC_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(s.p),
                               size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
        set_cuda_error(cudaErrorInvalidValue);
        return HGC_ERR_CUDA;
    }
    return HGC_OK;
}

bool rows_fit(const Strided &s)
{
    const long long most = 1ll << 39;  // bytes between rows that a copy can step over
    return (reinterpret_cast<uintptr_t>(s.p) & 15u) == 0 && s.row > 0 && s.head > 0 && s.row % 8 == 0 && s.head % 8 == 0 && s.row < most && s.head < most;
}

template <typename K> int launch(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const Args &a, const Maps &maps)
{
    HGC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    HGC_CUDA_TRY(launch_pdl(kernel, grid, threads, smem, stream, a, maps));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

template <typename T, int CHUNKS> int grad_queries_mma(const Args &a, const Maps &maps, cudaStream_t stream)
{
    using F = GradQueries<CHUNKS>;
    const dim3 grid((unsigned)tile_count(a.n_q, kMmaRows / a.pack, a.n_events), a.heads / a.pack, a.splits);
    return launch(grad_queries_mma_kernel<T, CHUNKS>, grid, kBlock, F::kSmem, stream, a, maps);
}
template <typename T, int CHUNKS> int grad_keys_mma(const Args &a, const Maps &maps, cudaStream_t stream)
{
    using F = GradKeys<CHUNKS>;
    const dim3 grid((unsigned)tile_count(a.n_k, kMmaRows, a.n_events), a.kv_heads, a.splits);
    return launch(grad_keys_mma_kernel<T, CHUNKS>, grid, F::kThreads, F::kSmem, stream, a, maps);
}

template <typename T, int CHUNKS> int forward_mma(const Args &a, const Maps &maps, cudaStream_t stream)
{
    const dim3 grid((unsigned)tile_count(a.n_q, kMmaRows / a.pack, a.n_events), a.heads / a.pack, a.splits);
    return launch(forward_mma_kernel<T, CHUNKS>, grid, kBlock, Forward<CHUNKS>::kSmem, stream, a, maps);
}

}  // namespace

bool mma_takes(const Args &a, int dtype)
{
    const auto aligned = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    return (dtype == HGC_FLOAT16 || dtype == HGC_BFLOAT16) && a.dim % 8 == 0 && a.n_q > 0 && a.n_k > 0 && rows_fit(a.q) && rows_fit(a.k) && rows_fit(a.v) &&
           aligned(a.to) && aligned(a.to2) && aligned(a.grad);
}

int mma_forward(const Args &a, int dtype, cudaStream_t stream)
{
    Maps maps;
    if (const int rc = map_of(&maps.q, a.q, dtype, a.dim, a.heads, a.n_q, a.pack, kMmaRows / a.pack)) return rc;
    if (const int rc = map_of(&maps.k, a.k, dtype, a.dim, a.kv_heads, a.n_k, 1, mma_keys(a.dim))) return rc;
    if (const int rc = map_of(&maps.v, a.v, dtype, a.dim, a.kv_heads, a.n_k, 1, mma_keys(a.dim))) return rc;
    if (dtype == HGC_FLOAT16) return a.dim <= 64 ? forward_mma<__half, 1>(a, maps, stream) : forward_mma<__half, 2>(a, maps, stream);
    return a.dim <= 64 ? forward_mma<__nv_bfloat16, 1>(a, maps, stream) : forward_mma<__nv_bfloat16, 2>(a, maps, stream);
}

int mma_grad_queries(const Args &a, int dtype, cudaStream_t stream)
{
    const Strided grad{a.grad, (long long)a.heads * a.dim, a.dim};
    Maps maps;
    if (const int rc = map_of(&maps.q, a.q, dtype, a.dim, a.heads, a.n_q, a.pack, kMmaRows / a.pack)) return rc;
    if (const int rc = map_of(&maps.grad, grad, dtype, a.dim, a.heads, a.n_q, a.pack, kMmaRows / a.pack)) return rc;
    if (const int rc = map_of(&maps.k, a.k, dtype, a.dim, a.kv_heads, a.n_k, 1, kMmaGradStep)) return rc;
    if (const int rc = map_of(&maps.v, a.v, dtype, a.dim, a.kv_heads, a.n_k, 1, kMmaGradStep)) return rc;
    if (dtype == HGC_FLOAT16) return a.dim <= 64 ? grad_queries_mma<__half, 1>(a, maps, stream) : grad_queries_mma<__half, 2>(a, maps, stream);
    return a.dim <= 64 ? grad_queries_mma<__nv_bfloat16, 1>(a, maps, stream) : grad_queries_mma<__nv_bfloat16, 2>(a, maps, stream);
}

int mma_grad_keys(const Args &a, int dtype, cudaStream_t stream)
{
    const Strided grad{a.grad, (long long)a.heads * a.dim, a.dim};
    Maps maps;
    if (const int rc = map_of(&maps.q, a.q, dtype, a.dim, a.heads, a.n_q, a.pack, kMmaGradStep / a.pack)) return rc;
    if (const int rc = map_of(&maps.grad, grad, dtype, a.dim, a.heads, a.n_q, a.pack, kMmaGradStep / a.pack)) return rc;
    if (const int rc = map_of(&maps.k, a.k, dtype, a.dim, a.kv_heads, a.n_k, 1, kMmaRows)) return rc;
    if (const int rc = map_of(&maps.v, a.v, dtype, a.dim, a.kv_heads, a.n_k, 1, kMmaRows)) return rc;
    if (dtype == HGC_FLOAT16) return a.dim <= 64 ? grad_keys_mma<__half, 1>(a, maps, stream) : grad_keys_mma<__half, 2>(a, maps, stream);
    return a.dim <= 64 ? grad_keys_mma<__nv_bfloat16, 1>(a, maps, stream) : grad_keys_mma<__nv_bfloat16, 2>(a, maps, stream);
}

}  // namespace attn
}  // namespace hgc
