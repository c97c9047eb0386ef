// Attention of a few queries per event, the new ones of a service say, to all of its keys: bound by reading keys and values once.
//
// A key has as many lanes as its row has 16-byte vectors, and up to eight rows of queries (tokens times heads that share the key
// head) are held in registers; every group of lanes goes through keys of its own with its own running maximum and sum, and all are
// joined at the end.  Tensor cores give a lane a row and would leave most lanes without one.  64 queries with a key head for each of
// their heads on 1.28M keys: 159 us for two key heads, 509 for eight, 5.1 TB/s.  With more rows the operations on them bound it.
#include "cross_attention.cuh"
#include "mma_device.cuh"

namespace hgc {
namespace attn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kFewRows = 8;
// Keys that a lane group takes in a step, and steps whose rows are in shared memory or on their way there.  A lane copies what it will
// read itself, so that nothing has to be waited for but its own copies.
template <int R> constexpr int kAhead = R == 8 ? 2 : 4;
constexpr int kStages = 3;
template <int R> constexpr int kStageBytes = kWarps * kAhead<R> * 2 * 32 * 16;
__device__ __forceinline__ void copy16(unsigned to, const void *from, bool in)  // zeros where not `in`
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}

template <typename T> constexpr int kVec = 16 / sizeof(T);
template <typename T> __device__ __forceinline__ void unpack(mma::pair (&to)[kVec<T> / 2], const uint4 &q)
{
    const unsigned u[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
        to[0] = mma::pair_of(__uint_as_float(u[0]), __uint_as_float(u[1]));
        to[1] = mma::pair_of(__uint_as_float(u[2]), __uint_as_float(u[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = mma::unpack2<T>(u[i]);
            to[i] = mma::pair_of(f.x, f.y);
        }
    }
}

template <typename T, int R>
__global__ void __launch_bounds__(kThreads, R == 8 ? 1 : 2)
few_kernel(const __grid_constant__ Args a, int lanes_log2)
{
    pdl_begin();
    constexpr int V = kVec<T>, H = V / 2, U = kAhead<R>;
    extern __shared__ __align__(16) float s_mem[];  // [kWarps][R][dim] sums, then [kWarps][R] maxima and [kWarps][R] sums of weights
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int tokens = R / a.pack, head0 = blockIdx.y * a.pack, kv = head0 / a.group;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_splits(a, t, kThreads);
    const Tile tile = find_tile(a.rs_q, a.n_q, a.n_events, tokens, blockIdx.x);
    if (tile.begin >= tile.end) return;
    const int n_rows = (tile.end - tile.begin) * a.pack;
    const int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    const int2 part = part_of(max(0, (keys.y - keys.x + kFewStep - 1) / kFewStep), blockIdx.z, a.splits);
    const int begin = keys.x + part.x * kFewStep, end = min(keys.y, keys.x + part.y * kFewStep);

    const int lanes = 1 << lanes_log2, groups = 32 >> lanes_log2, column = (lane & (lanes - 1)) * V, group = lane >> lanes_log2;
    const bool has = column < a.dim;
    const float c = a.scale * kLog2e;
    mma::pair q[R][H], acc[R][H];
    float top[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n_rows && has)
            v = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q.p) + (long long)(tile.begin + r / a.pack) * a.q.row +
                                                 (long long)(head0 + r % a.pack) * a.q.head + column);
        unpack<T>(q[r], v);
#pragma unroll
        for (int i = 0; i < H; i++) {
            q[r][i] = mma::mul2(q[r][i], mma::pair_of(c, c));
            acc[r][i] = 0;
        }
        top[r] = -INFINITY;
        sum[r] = 0.f;
    }
    const T *k_base = static_cast<const T *>(a.k.p) + (long long)kv * a.k.head + column;
    const T *v_base = static_cast<const T *>(a.v.p) + (long long)kv * a.v.head + column;
    // all lanes of a warp go through the loop together: groups meet in the sums over lanes
    const int stride = kWarps * groups * U, base = begin + warp * groups * U + group;
    const int steps = max(0, (end - (begin + warp * groups * U) + stride - 1) / stride);
    const unsigned ring = mma::smem_address(s_mem) + (warp * U * 2 * 32 + lane) * 16;
    unsigned seen_ahead[kStages] = {};  // of the steps on their way, a bit per key
    const auto ask = [&](int j, unsigned &seen) {
        seen = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int key = base + j * stride + u * groups;
            const bool in = j < steps && key < end;
            const unsigned to = ring + j % kStages * kStageBytes<R> + u * 2 * 32 * 16;
            copy16(to, k_base + (in ? (long long)key * a.k.row : 0), in && has);
            copy16(to + 32 * 16, v_base + (in ? (long long)key * a.v.row : 0), in && has);
            if (in && (a.mask == nullptr || a.mask[key] != 0)) seen |= 1u << u;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (steps > 0) {
#pragma unroll
        for (int j = 0; j < kStages - 1; j++) ask(j, seen_ahead[j]);
    }
    for (int j = 0; j < steps; j++) {
        ask(j + kStages - 1, seen_ahead[kStages - 1]);
        asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 1) : "memory");
        uint4 k_in[U], v_in[U];
        bool seen[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const unsigned from = ring + j % kStages * kStageBytes<R> + u * 2 * 32 * 16;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(k_in[u].x), "=r"(k_in[u].y), "=r"(k_in[u].z), "=r"(k_in[u].w) : "r"(from) : "memory");
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v_in[u].x), "=r"(v_in[u].y), "=r"(v_in[u].z), "=r"(v_in[u].w) : "r"(from + 32 * 16) : "memory");
            seen[u] = (seen_ahead[0] >> u) & 1u;
        }
#pragma unroll
        for (int i = 0; i + 1 < kStages; i++) seen_ahead[i] = seen_ahead[i + 1];
        float s[R][U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            mma::pair k[H];
            unpack<T>(k, k_in[u]);
#pragma unroll
            for (int r = 0; r < R; r++) {
                mma::pair dot = 0;
#pragma unroll
                for (int i = 0; i < H; i++) dot = mma::fma2(q[r][i], k[i], dot);
                const float2 d = mma::parts(dot);
                s[r][u] = d.x + d.y;
            }
        }
        for (int w = lanes >> 1; w > 0; w >>= 1)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int u = 0; u < U; u++) s[r][u] += __shfl_xor_sync(0xffffffffu, s[r][u], w);
        bool grown = false;
        float next[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            next[r] = top[r];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (!seen[u]) s[r][u] = -INFINITY;
                next[r] = fmaxf(next[r], s[r][u]);
            }
            grown = grown || next[r] > top[r];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float shrink = mma::exp2_fast(top[r] - (next[r] == -INFINITY ? 0.f : next[r]));
                top[r] = next[r];
                sum[r] *= shrink;
#pragma unroll
                for (int i = 0; i < H; i++) acc[r][i] = mma::mul2(acc[r][i], mma::pair_of(shrink, shrink));
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float from = top[r] == -INFINITY ? 0.f : top[r];
#pragma unroll
            for (int u = 0; u < U; u++) {
                s[r][u] = mma::exp2_fast(s[r][u] - from);
                sum[r] += s[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!seen[u]) v_in[u] = make_uint4(0, 0, 0, 0);  // whatever stands there
            mma::pair v[H];
            unpack<T>(v, v_in[u]);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < H; i++) acc[r][i] = mma::fma2(mma::pair_of(s[r][u], s[r][u]), v[i], acc[r][i]);
        }
    }
    // the groups of a warp
    for (int w = lanes; w < 32; w <<= 1)
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float other = __shfl_xor_sync(0xffffffffu, top[r], w), next = fmaxf(top[r], other), from = next == -INFINITY ? 0.f : next;
            const float mine = exp2f(top[r] - from), theirs = exp2f(other - from);
            top[r] = next;
            sum[r] = sum[r] * mine + __shfl_xor_sync(0xffffffffu, sum[r], w) * theirs;
#pragma unroll
            for (int i = 0; i < H; i++) {
                const float2 x = mma::parts(acc[r][i]);
                const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, x.x, w), __shfl_xor_sync(0xffffffffu, x.y, w));
                acc[r][i] = mma::pair_of(x.x * mine + y.x * theirs, x.y * mine + y.y * theirs);
            }
        }
    // the warps, in their order, where the rows were: those have been read, and the zeros asked for behind the last step are there too
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float *s_top = s_mem + kWarps * R * a.dim, *s_sum = s_top + kWarps * R;
    if (group == 0) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (has)
#pragma unroll
                for (int i = 0; i < H; i++)
                    *reinterpret_cast<float2 *>(s_mem + (warp * R + r) * a.dim + column + 2 * i) = mma::parts(acc[r][i]);
            if (lane == 0) {
                s_top[warp * R + r] = top[r];
                s_sum[warp * R + r] = sum[r];
            }
        }
    }
    __syncthreads();
    const long long all_rows = (long long)a.n_q * a.heads;
    for (int i = t; i < n_rows * a.dim; i += kThreads) {
        const int r = i / a.dim, d = i - r * a.dim;
        float most = -INFINITY, total = 0.f, o = 0.f;
        for (int w = 0; w < kWarps; w++) most = fmaxf(most, s_top[w * R + r]);
        const float from = most == -INFINITY ? 0.f : most;
        for (int w = 0; w < kWarps; w++) {
            const float f = exp2f(s_top[w * R + r] - from);
            total += s_sum[w * R + r] * f;
            o = fmaf(s_mem[(w * R + r) * a.dim + d], f, o);
        }
        const bool none = most == -INFINITY && total == 0.f;  // a maximum passes over what is no number, the sum does not
        o = none ? 0.f : o / total;
        const long long row = (long long)(tile.begin + r / a.pack) * a.heads + head0 + r % a.pack;
        if (a.splits > 1) a.part[(blockIdx.z * all_rows + row) * a.dim + d] = o;
        else store_rounded(static_cast<T *>(a.to) + row * a.dim + d, a.rest == nullptr ? nullptr : static_cast<T *>(a.rest) + row * a.dim + d, o);
        if (d == 0) (a.splits > 1 ? a.part_lse + blockIdx.z * all_rows : a.lse)[row] = none ? -INFINITY : most * kLn2 + logf(total);
    }
}

template <typename T, int R> int launch(const Args &a, int lanes_log2, cudaStream_t stream)
{
    const dim3 grid((unsigned)tile_count(a.n_q, R / a.pack, a.n_events), a.heads / a.pack, a.splits);
    const size_t joined = sizeof(float) * kWarps * R * (a.dim + 2), ring = (size_t)kStages * kStageBytes<R>, smem = joined > ring ? joined : ring;
    HGC_CUDA_TRY(cudaFuncSetAttribute(few_kernel<T, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    HGC_CUDA_TRY(launch_pdl(few_kernel<T, R>, grid, kThreads, smem, stream, a, lanes_log2));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}
template <typename T> int run(Args a, int rows, cudaStream_t stream)
{
    int lanes_log2 = 0;
    while ((kVec<T> << lanes_log2) < a.dim) lanes_log2++;
    if constexpr (sizeof(T) == 4)
        if (rows > 2) return rows <= 4 ? launch<T, 4>(a, lanes_log2, stream) : launch<T, 8>(a, lanes_log2, stream);
    return rows <= 1 ? launch<T, 1>(a, lanes_log2, stream) : launch<T, 2>(a, lanes_log2, stream);
}

}  // namespace

int few_pack(int group)
{
    int pack = group < kFewRows ? group : kFewRows;
    while (group % pack != 0) pack--;
    return pack;
}
int few_rows(int n_q, int n_events, int pack)
{
    const int some = n_events > 0 ? n_events : 1;
    const long long mean = n_q > 0 ? ((long long)n_q + some - 1) / some : 1, rows = mean * pack;
    return mean > kFewRows / pack ? 0 : rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
}
bool few_takes(const Args &a, int rows, int dtype)
{
    // 16-bit types: from four rows on the tensor cores are faster, though most of their rows are empty (64 queries on 1.28M keys, us there /
    // here: one row a block 224 / 159, four 224 / 260, eight 230 / 457).  Float32 has tiles of 64 rows on the other side (64 columns, the
    // same lengths, eight heads: a row a block 5664 / 814, four 1443 / 279, eight 669 / 381; 700 keys 55 / 44).
    if (rows == 0 || (rows > 2 && dtype != HGC_FLOAT32)) return false;
    const int bytes = dtype == HGC_FLOAT32 ? 4 : 2, vec = 16 / bytes;
    const auto fits = [&](const Strided &s) { return (reinterpret_cast<uintptr_t>(s.p) & 15u) == 0 && s.row % vec == 0 && s.head % vec == 0; };
    return a.dim % vec == 0 && a.n_k > 0 && fits(a.q) && fits(a.k) && fits(a.v);
}
int few_forward(const Args &a, int rows, int dtype, cudaStream_t stream)
{
    return dtype == HGC_FLOAT32 ? run<float>(a, rows, stream) : dtype == HGC_FLOAT16 ? run<__half>(a, rows, stream) : run<__nv_bfloat16>(a, rows, stream);
}

}  // namespace attn
}  // namespace hgc
