// Norm of the heads of queries and keys and their rotation by positions, in one pass over the rows, forward and backward.
//
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps) over a head's columns
//   the columns of an axis form pairs (a, b), of which pair i turns by t = position / base^(i / pairs):
//   y_a = n_a cos t - n_b sin t,  y_b = n_b cos t + n_a sin t;  columns behind the rotary ones stay as they are
//   backward: g = dy turned back,  dx = r (g w - x r^2 mean(g w x)),  dw = sum over rows and heads of g x r
//
// Bound by memory: a row is read once and written once.  A row belongs to as many lanes as it has 16-byte vectors (or pairs of columns,
// or columns, where it is not whole vectors).  The angle of
// a far position needs more digits than float32 has: its turns are counted in double and only their fraction is kept, once for all
// heads of a row (position * frequency in float32 is off by 0.06 rad at a million).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace hgc {
namespace {

constexpr int kMaxDim = 128;
constexpr int kMaxCount = 0x7fffffff - 8192;  // rows: a step past the end must not leave 32 bits
constexpr int kThreads = 256, kBlocksPerSm = 4;
constexpr int kMaxTokens = 64;  // rows of a block, whose angles are kept

// Where the partner of a column is.  The small numbers: that many columns further on in the same lane, for axes of few columns.
enum Pairs {
    kNeighbours = 1,  // columns 2 i and 2 i + 1
    kTwoOn = 2,
    kFourOn = 4,
    kHalves = 16,     // columns i and i + pairs, whole vectors apart: in two lanes
    kBothHalves = 17, // columns i and i + pairs, all that there are: a lane has a vector of either half
    kAnywhere = 18    // through shared memory
};

struct Set {
    const void *x, *weight, *positions, *grad;
    void *y;             // or the gradient of x
    float *weight_part;  // [blocks of the set, dim]
    long long row, head;
    int n, heads, weight_float, tokens, blocks;
};

struct Call {
    Set set[2];
    double turns[kMaxDim / 2];  // turns per unit of position
    int dim, rotary, axes, pairs, axis_factor, position_type, interleaved, lanes_log2;
    float eps;
};

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V columns at one address; a whole 16-byte vector, or two columns, or one
template <typename T, int V> struct Vec { alignas(V * sizeof(T)) T v[V]; };

// two columns at a time where they come in 32 bits
__device__ __forceinline__ float2 two(unsigned v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ float2 two(unsigned v, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ unsigned both(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&r);
}
__device__ __forceinline__ unsigned both(float a, float b, __half)
{
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&r);
}
template <typename T, int V>
__device__ __forceinline__ void to_floats(float (&to)[V], const Vec<T, V> &from)
{
    if constexpr (sizeof(T) == 2 && V == 8) {
        const uint4 q = *reinterpret_cast<const uint4 *>(&from);
        const unsigned u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = two(u[i], T{});
            to[2 * i] = f.x;
            to[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) to[i] = as_float(from.v[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store(T *__restrict__ to, const float (&from)[V])
{
    if constexpr (sizeof(T) == 2 && V == 8) {
        *reinterpret_cast<uint4 *>(to) = make_uint4(both(from[0], from[1], T{}), both(from[2], from[3], T{}), both(from[4], from[5], T{}),
                                                    both(from[6], from[7], T{}));
    } else {
        Vec<T, V> q;
#pragma unroll
        for (int i = 0; i < V; i++) q.v[i] = rounded<T>(from[i]);
        *reinterpret_cast<Vec<T, V> *>(to) = q;
    }
}

// Where the angle of a pair is in a row's part of the table.  Lanes read two angles at a time, 16 bytes; kept in the order of the
// lanes these do not meet in the same banks.
template <int V, Pairs P> __device__ __forceinline__ int place(int pair, int n_pairs)
{
    constexpr int A = P == kHalves || P == kBothHalves ? V : (V + 1) / 2;  // angles of a lane
    if constexpr (P == kAnywhere || A < 4) return pair;
    else return pair < n_pairs / A * A ? (pair % A / 2 * (n_pairs / A) + pair / A) * 2 + pair % 2 : pair;
}
// The angles of rows [first, first + n) of a set: (cos, sin) of every pair of columns.  The whole turns go in double: what is left is
// off by (5 + ln base) 2^-53 of the position's turns at most (the turns of a unit by the exponent i / pairs, ln base, the power, 2, the
// constant and the product, and the fraction).
template <typename T, int V, Pairs P>
__device__ __forceinline__ void angles(const Call &c, const Set &s, const double *__restrict__ turns, int first, int n, float2 *__restrict__ table)
{
    const int pairs = c.rotary / 2, step_t = kThreads / pairs, step_p = kThreads - step_t * pairs;
    int token = threadIdx.x / pairs, p = threadIdx.x - token * pairs;
    while (token < n) {
        const int axis = p * c.axis_factor >> 16;  // p / c.pairs
        const long long at = (long long)(first + token) * c.axes + axis;
        const double x = c.position_type == HGC_POSITION_FLOAT32 ? (double)static_cast<const float *>(s.positions)[at]
                       : c.position_type == HGC_POSITION_INT32 ? (double)static_cast<const int *>(s.positions)[at]
                                                               : (double)static_cast<const long long *>(s.positions)[at];
        const double turn = turns[p - axis * c.pairs];
        float2 cs;
        const float part = (float)fma(x, turn, -rint(x * turn));
        if constexpr (sizeof(T) == 4) {
            sincospif(2.f * part, &cs.y, &cs.x);
        } else {  // off by 2^-20 at most, where results are rounded to 2^-11 or less
            cs.y = __sinf(6.283185307f * part);
            cs.x = __cosf(6.283185307f * part);
        }
        table[token * pairs + place<V, P>(p, pairs)] = cs;
        token += step_t;
        p += step_p;
        if (p >= pairs) { p -= pairs; token++; }
    }
}

// What a lane knows about its columns.
template <int V, int E, Pairs P> struct Columns {
    int column[E];       // first of V, or -1
    int pair[E];         // its angle in a row of the table (kNeighbours, kHalves: that of the first column)
    bool turned[E];
    int at, step;        // where the lane's first two angles are, and from there to its next two
    bool whole;          // all of its columns turn
    int partner_lane;    // kHalves
    float sign;          // kHalves: of the sine

    __device__ __forceinline__ Columns(const Call &c, int lane_in_row, int lanes)
    {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = P == kBothHalves ? lane_in_row * V + c.pairs * e : (lane_in_row + lanes * e) * V;
            column[e] = d < c.dim ? d : -1;
            turned[e] = d < c.rotary;
            pair[e] = 0;
        }
        whole = column[0] >= 0 && column[0] + V <= c.rotary;
        partner_lane = lane_id();
        sign = 0.f;
        if constexpr (P == kBothHalves) pair[0] = lane_in_row * V;
        if constexpr (P < kHalves) pair[0] = max(column[0], 0) / 2;  // a lane's columns hold whole axes, or neighbours
        if constexpr (P == kHalves) {
            const int span = max(2 * c.pairs, 1), axis = max(column[0], 0) / span, off = max(column[0], 0) - axis * span;
            const bool second = off >= c.pairs;
            pair[0] = axis * c.pairs + (second ? off - c.pairs : off);
            sign = second ? 1.f : -1.f;
            if (turned[0] && column[0] >= 0) partner_lane += (second ? -c.pairs : c.pairs) / V;
        }
        constexpr int A = P == kHalves || P == kBothHalves ? V : (V + 1) / 2;
        const int n_pairs = c.rotary / 2;
        const bool in_order = A < 4 || pair[0] >= n_pairs / A * A;
        at = in_order ? pair[0] : pair[0] / A * 2;
        step = in_order ? 2 : n_pairs / A * 2;
    }
};

// Turns a row's columns by `direction` times its angles.  All lanes of a warp take part.
template <int V, int E, Pairs P>
__device__ __forceinline__ void turn(float (&v)[E][V], const Columns<V, E, P> &k, const Call &c, const float2 *__restrict__ table, float direction,
                                     float *__restrict__ row_buffer)
{
    if constexpr (P < kHalves) {
        // pair j of the lane: columns (j / P) 2 P + j % P and P further on
        if (k.turned[0] && k.column[0] >= 0) {
#pragma unroll
            for (int j = 0; j < V / 2; j++) {
                const int first = j / P * (2 * P) + j % P;
                if (!k.whole && k.column[0] + first >= c.rotary) break;
                const float2 cs = table[k.at + j / 2 * k.step + j % 2];
                const float a = v[0][first], b = v[0][first + P], sine = cs.y * direction;
                v[0][first] = a * cs.x - b * sine;
                v[0][first + P] = b * cs.x + a * sine;
            }
        }
    } else if constexpr (P == kBothHalves) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float2 cs = table[k.at + i / 2 * k.step + i % 2];
            const float a = v[0][i], b = v[1][i], sine = cs.y * direction;
            v[0][i] = a * cs.x - b * sine;
            v[1][i] = b * cs.x + a * sine;
        }
    } else if constexpr (P == kHalves) {
        float other[V];
#pragma unroll
        for (int i = 0; i < V; i++) other[i] = __shfl_sync(0xffffffffu, v[0][i], k.partner_lane);
        if (k.turned[0] && k.column[0] >= 0) {
            const float sign = direction * k.sign;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float2 cs = table[k.at + i / 2 * k.step + i % 2];
                v[0][i] = v[0][i] * cs.x + other[i] * (cs.y * sign);
            }
        }
    } else {
        __syncwarp();
#pragma unroll
        for (int e = 0; e < E; e++)
            if (k.column[e] >= 0) {
#pragma unroll
                for (int i = 0; i < V; i++) row_buffer[k.column[e] + i] = v[e][i];
            }
        __syncwarp();
        const int span = 2 * c.pairs;
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (!k.turned[e] || k.column[e] < 0) continue;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int d = k.column[e] + i;
                if (d >= c.rotary) break;
                const int axis = d / span, off = d - axis * span;
                const bool second = c.interleaved ? off & 1 : off >= c.pairs;
                const int p = axis * c.pairs + (c.interleaved ? off >> 1 : second ? off - c.pairs : off);
                const int step = c.interleaved ? 1 : c.pairs;
                const float2 cs = table[p];
                const float other = row_buffer[second ? d - step : d + step];
                v[e][i] = v[e][i] * cs.x + other * (second ? cs.y : -cs.y) * direction;
            }
        }
    }
}

__device__ __forceinline__ float row_sum(float v, int lanes)
{
#pragma unroll
    for (int w = 16; w > 0; w >>= 1)
        if (w < lanes) v += __shfl_xor_sync(0xffffffffu, v, w);
    return v;
}

// A block has the rows of some tokens, with all their heads, kRows for every group of lanes that share a row; all of them are asked
// for before the angles are worked out, which takes as long as they are on their way.  It goes on with every blocks-th such group of
// tokens: what a block works out about its columns would cost as much as four rows of every lane do, and in the backward pass the
// sums for the gradient of the weights stay in registers.
constexpr int kRows = 2;
// blocks that a multiprocessor has registers for
template <int E, Pairs P, bool BACKWARD> constexpr int kResident = P == kAnywhere || (E > 1 && BACKWARD) ? 2 : BACKWARD || E > 1 ? 3 : kBlocksPerSm;
template <typename T, int V, int E, Pairs P, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, kResident<E, P, BACKWARD>)
norm_rotate_kernel(const __grid_constant__ Call c)
{
    pdl_begin();
    extern __shared__ __align__(16) float s_mem[];
    const bool second = (int)blockIdx.x >= c.set[0].blocks;
    const Set s = c.set[second];
    const int block = blockIdx.x - (second ? c.set[0].blocks : 0);
    float2 *s_table = reinterpret_cast<float2 *>(s_mem);
    const int lanes = 1 << c.lanes_log2, lane_in_row = threadIdx.x & (lanes - 1), sub = threadIdx.x >> c.lanes_log2, subs = kThreads >> c.lanes_log2;
    float *row_buffer = s_mem + s.tokens * c.rotary + sub * c.dim;  // kAnywhere
    const Columns<V, E, P> k(c, lane_in_row, lanes);
    const bool turns = c.rotary > 0 && s.positions != nullptr;
    __shared__ double s_turns[kMaxDim / 2];  // lanes that ask the arguments for different ones are served one after the other
    if (turns && threadIdx.x < c.pairs) s_turns[threadIdx.x] = c.turns[threadIdx.x];
    __syncthreads();
    float w[E][V], dw[E][V];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const bool in = k.column[e] >= 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            dw[e][i] = 0.f;
            w[e][i] = !in ? 0.f : s.weight == nullptr ? 1.f : s.weight_float ? static_cast<const float *>(s.weight)[k.column[e] + i]
                                                                              : as_float(static_cast<const T *>(s.weight)[k.column[e] + i]);
        }
    }
    const int groups = (s.n + s.tokens - 1) / s.tokens, token0 = sub / s.heads, head0 = sub - token0 * s.heads;
    const int step_t = subs / s.heads, step_h = subs - step_t * s.heads;
    const float inv_dim = 1.f / (float)c.dim;
    for (int group = block; group < groups; group += s.blocks) {
        const int first = group * s.tokens, n = min(s.tokens, s.n - first), rows = n * s.heads;
        if (turns && group != block) __syncthreads();  // the last group's angles have been read
        bool angles_due = turns;
        int token = token0, head = head0;
        for (int base = 0; base < rows; base += kRows * subs) {
            Vec<T, V> x_in[kRows][E], g_in[BACKWARD ? kRows : 1][E];
            int token_of[kRows];
            long long dense[kRows];
#pragma unroll
            for (int j = 0; j < kRows; j++) {
                const bool valid = base + j * subs + sub < rows;
                token_of[j] = valid ? token : -1;
                dense[j] = ((long long)(first + token) * s.heads + head) * c.dim;
                const T *x = static_cast<const T *>(s.x) + (long long)(first + token) * s.row + head * s.head;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    x_in[j][e] = Vec<T, V>{};
                    if (valid && k.column[e] >= 0) x_in[j][e] = *reinterpret_cast<const Vec<T, V> *>(x + k.column[e]);
                    if constexpr (BACKWARD) {
                        g_in[j][e] = Vec<T, V>{};
                        if (valid && k.column[e] >= 0) g_in[j][e] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(s.grad) + dense[j] + k.column[e]);
                    }
                }
                token += step_t;
                head += step_h;
                if (head >= s.heads) { head -= s.heads; token++; }
            }
            if (angles_due) {
                angles<T, V, P>(c, s, s_turns, first, n, s_table);
                __syncthreads();
                angles_due = false;
            }
#pragma unroll
            for (int j = 0; j < kRows; j++) {
                if (base + j * subs >= rows) break;  // for all lanes alike
                const bool valid = token_of[j] >= 0;
                float x[E][V], sum = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) to_floats<T, V>(x[e], x_in[j][e]);
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int i = 0; i < V; i++) sum = fmaf(x[e][i], x[e][i], sum);
                const float r = rsqrtf(row_sum(sum, lanes) * inv_dim + c.eps);
                const float2 *table = s_table + (valid ? token_of[j] : 0) * (c.rotary / 2);
                T *to = static_cast<T *>(s.y) + dense[j];
                if constexpr (!BACKWARD) {
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int i = 0; i < V; i++) x[e][i] = x[e][i] * r * w[e][i];
                    if (turns) turn<V, E, P>(x, k, c, table, 1.f, row_buffer);
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (valid && k.column[e] >= 0) store<T, V>(to + k.column[e], x[e]);
                } else {
                    float g[E][V], dot = 0.f;
#pragma unroll
                    for (int e = 0; e < E; e++) to_floats<T, V>(g[e], g_in[j][e]);
                    if (turns) turn<V, E, P>(g, k, c, table, -1.f, row_buffer);
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            if (valid) dw[e][i] = fmaf(g[e][i], x[e][i] * r, dw[e][i]);
                            g[e][i] *= w[e][i];
                            dot = fmaf(g[e][i], x[e][i], dot);
                        }
                    const float mean = row_sum(dot, lanes) * inv_dim * r * r;
#pragma unroll
                    for (int e = 0; e < E; e++) {
#pragma unroll
                        for (int i = 0; i < V; i++) g[e][i] = r * (g[e][i] - x[e][i] * mean);
                        if (valid && k.column[e] >= 0) store<T, V>(to + k.column[e], g[e]);
                    }
                }
            }
        }
    }
    if (BACKWARD && s.weight_part != nullptr) {
        // the block's sums, sub-row by sub-row in a fixed order
        float *s_dw = s_mem;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++)
            if (k.column[e] >= 0) {
#pragma unroll
                for (int i = 0; i < V; i++) s_dw[sub * c.dim + k.column[e] + i] = dw[e][i];
            }
        __syncthreads();
        for (int d = threadIdx.x; d < c.dim; d += kThreads) {
            float sum = 0.f;
            for (int i = 0; i < subs; i++) sum += s_dw[i * c.dim + d];
            s.weight_part[(long long)block * c.dim + d] = sum;
        }
    }
}

// Gradient of a set's weights from the blocks' sums, in double: a block per column.
struct Join {
    const float *part[2];
    void *to[2];
    int blocks[2], as_float[2];
};
template <typename T>
__global__ void __launch_bounds__(kThreads)
join_weights_kernel(const __grid_constant__ Join j, int dim)
{
    pdl_begin();
    __shared__ double s_sum[kThreads / 32];
    const int set = blockIdx.y, d = blockIdx.x;
    if (j.to[set] == nullptr) return;
    double sum = 0.;
    for (int i = threadIdx.x; i < j.blocks[set]; i += kThreads) sum += j.part[set][(long long)i * dim + d];
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    if (lane_id() == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.;
        for (int i = 0; i < kThreads / 32; i++) sum += s_sum[i];
        if (j.as_float[set]) static_cast<float *>(j.to[set])[d] = (float)sum;
        else static_cast<T *>(j.to[set])[d] = rounded<T>((float)sum);
    }
}

// -------------------------------------------------------------------------------------------------------------- host
int log2_up(int n)
{
    int b = 0;
    while ((1 << b) < n) b++;
    return b;
}

// Blocks that a set's gradient is summed in, at most.
int gradient_blocks(int n) { return (int)(n < kBlocksPerSm * (long long)sm_count() + 1 ? n : kBlocksPerSm * sm_count() + 1); }

template <typename T, int V, int E, Pairs P, bool BACKWARD>
int run(Call &c, cudaStream_t stream)
{
    // As many blocks as the chip holds at a time, shared by the sets according to their work: an angle takes about as long as four
    // elements, and is worked out once for all heads (8 and 2 heads of 64, blocks shared by rows 409 us, by work 253).
    long long groups[2], room = kResident<E, P, BACKWARD> * (long long)sm_count();
    double work[2];
    for (int i = 0; i < 2; i++) {
        const Set &s = c.set[i];
        groups[i] = s.n > 0 ? div_up(s.n, s.tokens) : 0;
        work[i] = (double)s.n * ((double)s.heads * c.dim + (s.positions != nullptr ? 2. * c.rotary : 0.));
    }
    for (int i = 0; i < 2; i++) {
        const long long share = groups[0] + groups[1] <= room ? groups[i] : (long long)(work[i] / (work[0] + work[1]) * (double)(room - 1)) + 1;
        c.set[i].blocks = (int)(share < groups[i] ? share : groups[i]);
    }
    const int subs = kThreads >> c.lanes_log2;
    const int tokens = c.set[0].tokens > c.set[1].tokens ? c.set[0].tokens : c.set[1].tokens;
    size_t smem = sizeof(float) * (size_t)(tokens * c.rotary + (P == kAnywhere ? subs * c.dim : 0));
    if (BACKWARD && smem < sizeof(float) * subs * c.dim) smem = sizeof(float) * subs * c.dim;
    const auto kernel = norm_rotate_kernel<T, V, E, P, BACKWARD>;
    HGC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    HGC_CUDA_TRY(launch_pdl(kernel, c.set[0].blocks + c.set[1].blocks, kThreads, smem, stream, c));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

template <typename T, bool BACKWARD>
int run_type(Call &c, cudaStream_t stream)
{
    constexpr int V = 16 / sizeof(T);
    const auto fits = [&](int v) {
        bool all = c.dim % v == 0;
        const auto aligned = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (v * sizeof(T)) == 0; };
        for (const Set &s : c.set)
            if (s.n > 0) all = all && aligned(s.x) && aligned(s.y) && s.row % v == 0 && s.head % v == 0 && (!BACKWARD || aligned(s.grad));
        return all;
    };
    const bool whole = fits(V), twos = !whole && fits(2);
    // a vector of either half to a lane, where the lanes of a row are then a power of two and all columns turn together
    const bool both = whole && !c.interleaved && c.axes == 1 && c.rotary == c.dim && c.dim % (2 * V) == 0 && (c.dim & (c.dim - 1)) == 0;
    c.lanes_log2 = both ? log2_up(c.dim / V) - 1 : log2_up(c.dim / (whole ? V : twos ? 2 : 1));
    if (c.lanes_log2 > 5) c.lanes_log2 = 5;
    const int subs = kThreads >> c.lanes_log2;
    for (Set &s : c.set) {
        // about four rows for every group of lanes, which share the angles; fewer where that leaves multiprocessors without a block
        const long long even = ((long long)c.set[0].n * c.set[0].heads + (long long)c.set[1].n * c.set[1].heads) / (2LL * sm_count() * subs);
        const int each = even < 1 ? 1 : even > 4 ? 4 : (int)even;
        const int tokens = s.heads > 0 ? each * subs / s.heads : 1;
        s.tokens = tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens;
    }
    // Two columns at a time, or one, where rows are not whole vectors, with as many per lane as the width needs (288k rows of 4 heads of 22 in
    // bf16, forward and backward, always four single columns a lane: 1120 us, so 560).
    if (twos) {
        if (c.dim > 64) return run<T, 2, 2, kAnywhere, BACKWARD>(c, stream);
        if (c.interleaved || c.pairs == 1) return run<T, 2, 1, kNeighbours, BACKWARD>(c, stream);
        return c.pairs % 2 == 0 ? run<T, 2, 1, kHalves, BACKWARD>(c, stream) : run<T, 2, 1, kAnywhere, BACKWARD>(c, stream);
    }
    if (!whole)
        return c.dim <= 32 ? run<T, 1, 1, kAnywhere, BACKWARD>(c, stream)
             : c.dim <= 64 ? run<T, 1, 2, kAnywhere, BACKWARD>(c, stream) : run<T, 1, 4, kAnywhere, BACKWARD>(c, stream);
    if (both) return run<T, V, 2, kBothHalves, BACKWARD>(c, stream);
    if (c.interleaved) return run<T, V, 1, kNeighbours, BACKWARD>(c, stream);
    if (c.rotary == 0 || c.pairs % V == 0) return run<T, V, 1, kHalves, BACKWARD>(c, stream);
    if (c.pairs == 1) return run<T, V, 1, kNeighbours, BACKWARD>(c, stream);
    if (c.pairs == 2) return run<T, V, 1, kTwoOn, BACKWARD>(c, stream);
    if constexpr (V == 8)
        if (c.pairs == 4) return run<T, V, 1, kFourOn, BACKWARD>(c, stream);
    return run<T, V, 1, kAnywhere, BACKWARD>(c, stream);
}

template <typename T> int join_weights(const Join &j, int dim, cudaStream_t stream)
{
    HGC_CUDA_TRY(launch_pdl(join_weights_kernel<T>, dim3(dim, 2), kThreads, 0, stream, j, dim));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

int check(const hgc_norm_rotate_rows *sets, int n_sets, int dim, int rotary_dim, int n_axes, int position_type, double base, float eps, int dtype, bool backward)
{
    if (sets == nullptr || n_sets < 1 || n_sets > 2 || dim < 1 || rotary_dim < 0 || rotary_dim > dim || n_axes < 1 || rotary_dim % (2 * n_axes) != 0 ||
        position_type < HGC_POSITION_FLOAT32 || position_type > HGC_POSITION_INT64 || !(base > 1.) || !(base < 1e30) || !(eps >= 0.f) ||
        dtype < 0 || dtype > HGC_BFLOAT16)
        return HGC_ERR_INVALID_ARGUMENT;
    if (dim > kMaxDim) return HGC_ERR_UNSUPPORTED;
    for (int i = 0; i < n_sets; i++) {
        const hgc_norm_rotate_rows &s = sets[i];
        if (s.n < 0 || s.n_heads < 1 || s.row_stride < 0 || s.head_stride < 0) return HGC_ERR_INVALID_ARGUMENT;
        if (s.n > kMaxCount || s.n_heads > 65535) return HGC_ERR_UNSUPPORTED;
        if (s.n > 0 && (!s.d_x || (!backward && !s.d_y) || (backward && (!s.d_grad_y || !s.d_grad_x)))) return HGC_ERR_INVALID_ARGUMENT;
        if (s.d_weight && s.weight_type != HGC_FLOAT32 && s.weight_type != dtype) return HGC_ERR_INVALID_ARGUMENT;
        if (backward && s.d_grad_weight && !s.d_weight) return HGC_ERR_INVALID_ARGUMENT;
    }
    return HGC_OK;
}

Call call_of(const hgc_norm_rotate_rows *sets, int n_sets, int dim, int rotary_dim, int n_axes, int position_type, int interleaved, double base, float eps,
             bool backward)
{
    Call c = {};
    c.dim = dim; c.rotary = rotary_dim; c.axes = n_axes; c.pairs = rotary_dim / (2 * n_axes);
    c.position_type = position_type; c.interleaved = interleaved; c.eps = eps;
    if (c.pairs > 0) {
        c.axis_factor = 65536 / c.pairs + 1;  // exact for the up to 64 pairs of a row
        // each for itself: a product that is carried on is off by 2^-47 after 63 steps, which a far position makes an angle of
        for (int i = 0; i < c.pairs; i++) c.turns[i] = 0.15915494309189533577 * pow(base, -(double)i / c.pairs);  // turns of a radian
    }
    for (int i = 0; i < n_sets; i++) {
        Set &s = c.set[i];
        s.x = sets[i].d_x; s.weight = sets[i].d_weight; s.positions = sets[i].d_positions;
        s.grad = sets[i].d_grad_y; s.y = backward ? sets[i].d_grad_x : sets[i].d_y;
        s.row = sets[i].row_stride; s.head = sets[i].head_stride;
        s.n = sets[i].n; s.heads = sets[i].n_heads;
        s.weight_float = sets[i].weight_type == HGC_FLOAT32;
    }
    return c;
}

}  // namespace
}  // namespace hgc

using namespace hgc;

extern "C" int hgc_norm_rotate(const hgc_norm_rotate_rows *sets, int n_sets, int dim, int rotary_dim, int n_axes, int position_type, int interleaved,
                               double base, float eps, int dtype, hgc_stream_t stream_)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (const int rc = check(sets, n_sets, dim, rotary_dim, n_axes, position_type, base, eps, dtype, false)) return rc;
    Call c = call_of(sets, n_sets, dim, rotary_dim, n_axes, position_type, interleaved, base, eps, false);
    if (c.set[0].n == 0 && c.set[1].n == 0) return HGC_OK;
    return dtype == HGC_FLOAT32 ? run_type<float, false>(c, stream)
         : dtype == HGC_FLOAT16 ? run_type<__half, false>(c, stream) : run_type<__nv_bfloat16, false>(c, stream);
}

extern "C" size_t hgc_norm_rotate_grad_workspace_bytes(const hgc_norm_rotate_rows *sets, int n_sets, int dim)
{
    if (sets == nullptr || n_sets < 1 || n_sets > 2 || dim < 1 || dim > kMaxDim) return 0;
    Sizer z;
    for (int i = 0; i < n_sets; i++) {
        if (sets[i].n < 0 || sets[i].n_heads < 1) return 0;
        z.take<float>((size_t)gradient_blocks(sets[i].n) * dim);
    }
    return z.used;
}

extern "C" int hgc_norm_rotate_grad(const hgc_norm_rotate_rows *sets, int n_sets, int dim, int rotary_dim, int n_axes, int position_type, int interleaved,
                                    double base, float eps, int dtype, void *workspace, size_t workspace_bytes, hgc_stream_t stream_)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (const int rc = check(sets, n_sets, dim, rotary_dim, n_axes, position_type, base, eps, dtype, true)) return rc;
    if (const int rc = check_workspace(workspace, workspace_bytes, hgc_norm_rotate_grad_workspace_bytes(sets, n_sets, dim))) return rc;
    Call c = call_of(sets, n_sets, dim, rotary_dim, n_axes, position_type, interleaved, base, eps, true);
    Carver carver(workspace);
    Join j = {};
    bool join = false;
    for (int i = 0; i < n_sets; i++) {
        Set &s = c.set[i];
        float *part = carver.take<float>((size_t)gradient_blocks(s.n) * dim);
        s.weight_part = sets[i].d_grad_weight ? part : nullptr;
        j.part[i] = part;
        j.to[i] = sets[i].d_grad_weight;
        j.as_float[i] = s.weight_float;
        join = join || j.to[i] != nullptr;
    }
    if (c.set[0].n > 0 || c.set[1].n > 0) {
        if (const int rc = dtype == HGC_FLOAT32 ? run_type<float, true>(c, stream)
                         : dtype == HGC_FLOAT16 ? run_type<__half, true>(c, stream) : run_type<__nv_bfloat16, true>(c, stream))
            return rc;
    }
    if (!join) return HGC_OK;
    for (int i = 0; i < 2; i++) j.blocks[i] = c.set[i].n > 0 ? c.set[i].blocks : 0;
    return dtype == HGC_FLOAT32 ? join_weights<float>(j, dim, stream)
         : dtype == HGC_FLOAT16 ? join_weights<__half>(j, dim, stream) : join_weights<__nv_bfloat16>(j, dim, stream);
}
