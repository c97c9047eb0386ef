// Attention between two ragged sets of rows on the tensor cores, for 16-bit types.
//
// Blocks of twenty warps have a multiprocessor each.  Sixteen of them do the elementwise work on rows of tensor memory (with eight,
// each instruction of a warp waited for the one before, and none of the units was half busy), four keep them fed: copies, products
// of scores, products of sums, rows to clear.  They meet at barriers in shared memory only.
#include <cuda.h>
#include <atomic>

#include "cross_attention.cuh"
#include "mma_device.cuh"

namespace hgc {
namespace attn {
namespace {

using namespace mma;

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
        const bool in = key < n && (mask == nullptr || fresh(mask + k0 + key) != 0);
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

// Where the lanes' rows of a result begin.  Two lanes write a row together, 32 bytes of it: stores of 16 bytes to 32 rows each took
// twice as long.
struct Rows {
    long long at, other;
    bool store, store_other;
    __device__ __forceinline__ Rows(long long begin, bool in) : at(begin), store(in)
    {
        other = __shfl_xor_sync(0xffffffffu, at, 1);
        store_other = __shfl_xor_sync(0xffffffffu, (int)in, 1) != 0;
    }
};
// 16 columns of a row of a result; all lanes of a warp call this.  rest: for what the rounding leaves, or null.
template <typename T>
__device__ __forceinline__ void store16(void *to, void *rest, float *part, const Rows &rows, int d, int dim, const unsigned (&v)[16], float factor)
{
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = __uint_as_float(v[i]) * factor;
    if (part != nullptr) {
        float4 *p = reinterpret_cast<float4 *>(part + rows.at + d);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (rows.store && d + 4 * i < dim) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
#pragma unroll 1
        for (void *next = to;; next = rest) {
            unsigned h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
            const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
            // first the even lanes' rows: they keep their first 16 bytes and give away the second; then the odd ones'
            const bool odd = lane_id() & 1;
            const uint4 give = odd ? a : b;
            const uint4 got = make_uint4(__shfl_xor_sync(0xffffffffu, give.x, 1), __shfl_xor_sync(0xffffffffu, give.y, 1),
                                         __shfl_xor_sync(0xffffffffu, give.z, 1), __shfl_xor_sync(0xffffffffu, give.w, 1));
            T *const base = static_cast<T *>(next) + d + (odd ? 8 : 0);
            if (d + (odd ? 8 : 0) < dim) {
                if (odd ? rows.store_other : rows.store) *reinterpret_cast<uint4 *>(base + (odd ? rows.other : rows.at)) = odd ? got : a;
                if (odd ? rows.store : rows.store_other) *reinterpret_cast<uint4 *>(base + (odd ? rows.at : rows.other)) = odd ? b : got;
            }
            if (rest == nullptr || next == rest) break;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 there = unpack2<T>(h[i]);
                x[2 * i] -= there.x;
                x[2 * i + 1] -= there.y;
            }
        }
    }
}

// A tile is twice 128 rows of queries of an event, each half with eight warps that do its softmax (half a row per lane); it goes
// through the keys of the event, kKeys a step.  Scores S = Q K^T and, in their place, weights P (16 bits) are in buffers of tensor memory that
// the halves use in turn, so that the next scores are done when a softmax ends; the sums O = P V lie beside them.  Four more warps
// copy queries, keys and values, issue scores, issue sums, and clear what must not be summed.
//
// Where events have no more than 128 rows, `alternate`, a tile is 128 rows, and the two times eight warps take its steps in turn, each
// with sums of their own: twice as many parts to join (64 queries on 1.28M keys 250 -> 224 us).
//
// A block takes one tile after the other from a counter, and every warp goes on to the next tile as soon as its own part is done: copies
// and scores of a tile run under the softmax and the results of the one before.  With a tile per block, 371k queries on 1152 keys
// took 490 us, two thirds of them for starting and ending blocks.
template <int CHUNKS> struct Forward {
    static constexpr int kKeys = CHUNKS == 1 ? 128 : 64, kStages = 4, kQueries = CHUNKS == 1 ? 2 : 1, kThreads = 640;
    static constexpr int kTileBytes = kKeys * kTile * CHUNKS, kHalfBytes = kMmaRows * kTile * CHUNKS, kQueryBytes = 2 * kHalfBytes;
    static constexpr int kBuffers = CHUNKS == 1 ? 3 : 4, kOut = kKeys * kBuffers, kColumns = 512, kItems = 4;
    static constexpr int kTiles = kQueries * kQueryBytes + 2 * kStages * kTileBytes;
    static constexpr int kBarriers = 3 + 3 * kStages + 3 * kBuffers + 2 * kQueries + 3 * kItems + 4 + 8;
    static constexpr int kBias = 512, kMaxAt = kBias + kStages * kKeys * 4, kItemAt = kMaxAt + 2 * 3 * 2 * kMmaRows * 4,
                         kSmem = kTiles + kItemAt + kItems * 48;  // behind the tiles
    static_assert(kOut + 128 * CHUNKS <= kColumns && 8 * kBarriers + 8 + 4 * kStages <= kBias && kSmem <= 232448, "room");
};

// What the warps of a block have to know of a tile; steps < 0: there is none any more.
struct Item {
    int steps, first, keys_end, dirty;  // of keys; steps from `dirty` on have some that are masked, or of another event
    int begin, end, head0, split;       // of queries
};

// Weights are held 2^kShift times as large as they are next to the row's scale, and that may lag behind the row's maximum by a factor
// of 2^kGrowth before the sums are scaled again.  Half precision reaches from 2^15 down to 2^-24 only, and many keys far below one that
// dominates have a share together: what is rounded away of n of them is n 2^-37 of the largest value (without a shift, one key
// 17.5 above 400k others took all of their 1 %).  2^14 and 2^1 cost wide heads 10 %: 128 columns, 200k queries on 1000 keys 545 -> 600 us.
template <typename T> struct Weights { static constexpr float kShift = 0.f, kGrowth = 8.f; };
template <> struct Weights<__half> { static constexpr float kShift = 12.f, kGrowth = 3.f; };

// Counts through rounds of N.
template <int N> struct Ring {
    int at = 0;
    unsigned turn = 0;
    __device__ __forceinline__ void go(int by)  // at most N
    {
        at += by;
        if (at >= N) at -= N, turn ^= 1;
    }
};

// REST: what the rounding of the results leaves is kept too; with that in every call, 1000 queries on 400k masked
// keys, 8 heads of 32, took 685 us, not 655.
template <typename T, int CHUNKS, bool REST>
__global__ void __launch_bounds__(Forward<CHUNKS>::kThreads, 1)
forward_mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps, int n_tiles, int n_items, int alternate)
{
    pdl_begin();
    using F = Forward<CHUNKS>;
    constexpr int N = F::kKeys, W = N / 32, B = F::kBuffers;
    extern __shared__ __align__(1024) char s_raw[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int tokens = kMmaRows / a.pack;  // of half a tile
    if (blockIdx.x == 0) check_splits(a, t, F::kThreads);

    const unsigned s_q = smem_address(s_raw), s_k = s_q + F::kQueries * F::kQueryBytes, s_v = s_k + F::kStages * F::kTileBytes;
    const unsigned bar = s_q + F::kTiles, scores_done = bar, sums_done = bar + 8, go = bar + 16, full = bar + 24, empty = full + 8 * F::kStages,
                   clean = empty + 8 * F::kStages, s_full = clean + 8 * F::kStages, p_full = s_full + 8 * B, used = p_full + 8 * B,
                   q_full = used + 8 * B, q_empty = q_full + 8 * F::kQueries, item_full = q_empty + 8 * F::kQueries,
                   item_empty = item_full + 8 * F::kItems, o_full = item_empty + 8 * F::kItems, o_empty = o_full + 16,
                   item_done = o_empty + 16, meet = item_done + 8 * F::kItems;
    unsigned *s_tmem = reinterpret_cast<unsigned *>(s_raw + F::kTiles + 8 * F::kBarriers);
    volatile int *gave_up = reinterpret_cast<volatile int *>(s_tmem + 1);
    volatile int *s_any = gave_up + 1;  // [kStages], whether a key of a step that is not whole is seen
    float *s_bias = reinterpret_cast<float *>(s_raw + F::kTiles + F::kBias);  // [kStages][kKeys], 0 or minus infinity
    Item *s_item = reinterpret_cast<Item *>(s_raw + F::kTiles + F::kItemAt);
    if (t == 0) {
        for (int i = 0; i < F::kBarriers; i++) {
            const unsigned at = bar + 8 * i;
            // arrivals: a half's warps; or of an item, all that read it: sixteen of the halves, and three
            barrier_init(at, at >= meet ? 2 : (at >= p_full && at < used) || at >= o_empty ? 8 : at >= item_empty && at < o_full ? 19 : 1);
        }
        barrier_init_done();
        *gave_up = 0;
    }
    if (warp == 19) tmem_alloc(s_tmem, F::kColumns);
    before_sync();
    __syncthreads();
    after_sync();
    const unsigned tmem = *s_tmem;

    if (warp == 16) {
        Ring<F::kItems> item;
        Ring<F::kStages> kv;
        Ring<F::kQueries> q;
        int k_copies = 0, q_copies = 0, taken = 0;
        bool ok = true;
        for (int next = blockIdx.x; ok;) {
            // the next tile that has rows
            Item it;
            it.steps = -1;
            while (next < n_items) {
                const int rest = next / n_tiles, split = rest / (a.heads / a.pack);
                const Tile tile = find_tile(a.rs_q, a.n_q, a.n_events, alternate ? tokens : 2 * tokens, next - rest * n_tiles);
                if (n_items > gridDim.x) {
                    if (lane == 0) next = gridDim.x + atomicAdd(a.counter, 1);
                    next = __shfl_sync(0xffffffffu, next, 0);
                } else {
                    next = n_items;
                }
                if (tile.begin >= tile.end) continue;
                const int2 keys = rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
                const int2 part = part_of(max(0, (keys.y - keys.x + N - 1) / N), split, a.splits);
                it.steps = part.y - part.x;
                it.first = keys.x + part.x * N;
                it.keys_end = keys.y;
                it.dirty = a.mask != nullptr ? 0 : min(it.steps, (keys.y - it.first) / N);
                it.begin = tile.begin;
                it.end = tile.end;
                it.head0 = (rest - split * (a.heads / a.pack)) * a.pack;
                it.split = split;
                break;
            }
            if (taken >= F::kItems) ok = wait_warp<true>(item_empty + 8 * item.at, item.turn ^ 1, gave_up, a.status);
            if (!ok) break;
            if (lane == 0) {
                s_item[item.at] = it;
                arrive(item_full + 8 * item.at);
            }
            __syncwarp();
            item.go(1);
            taken++;
            if (it.steps < 0) break;
            if (it.steps > 0 && elect()) {
                const int groups = it.end - it.begin > tokens ? 2 : 1, kv_head = it.head0 / a.group;
                if (q_copies >= F::kQueries) ok = wait(q_empty + 8 * q.at, q.turn ^ 1, gave_up, a.status);
                if (ok) {
                    arrive_expect(q_full + 8 * q.at, groups * CHUNKS * kTile * a.pack * tokens);
                    for (int g = 0; g < groups; g++)
                        for (int c = 0; c < CHUNKS; c++)
                            copy_box(s_q + q.at * F::kQueryBytes + g * F::kHalfBytes + c * kMmaRows * kTile, &maps.q, q_full + 8 * q.at, 64 * c, it.head0,
                                     it.begin + g * tokens);
                    q_copies++;
                    q.go(1);
                }
                for (int j = 0; j < it.steps && ok; j++) {
                    if (k_copies >= F::kStages) ok = wait(empty + 8 * kv.at, kv.turn ^ 1, gave_up, a.status);
                    if (!ok) break;
                    arrive_expect(full + 8 * kv.at, 2 * F::kTileBytes);
                    for (int c = 0; c < CHUNKS; c++) {
                        copy_box(s_k + kv.at * F::kTileBytes + c * N * kTile, &maps.k, full + 8 * kv.at, 64 * c, kv_head, it.first + j * N);
                        copy_box(s_v + kv.at * F::kTileBytes + c * N * kTile, &maps.v, full + 8 * kv.at, 64 * c, kv_head, it.first + j * N);
                    }
                    k_copies++;
                    kv.go(1);
                }
            }
            __syncwarp();  // the counts are the elected thread's, which is the same one every time
            ok = __all_sync(0xffffffffu, ok);
        }
        if (elect()) {  // no copy is under way when the block leaves
            for (int i = 0; i < min(q_copies, F::kQueries); i++) {
                if (--q.at < 0) q.at = F::kQueries - 1, q.turn ^= 1;
                drain(q_full + 8 * q.at, q.turn);
            }
            for (int i = 0; i < min(k_copies, F::kStages); i++) {
                if (--kv.at < 0) kv.at = F::kStages - 1, kv.turn ^= 1;
                drain(full + 8 * kv.at, kv.turn);
            }
        }
        __syncwarp();
    } else if (warp == 17) {
        if (elect()) {
            const int depth = (a.dim + 15) / 16;
            const unsigned shape_s = shape<T>(N, false);
            Ring<F::kItems> item;
            Ring<F::kStages> kv;
            Ring<F::kQueries> q;
            Ring<B> buffer;
            int scored = 0;
            unsigned clean_turns = 0;  // a bit per stage: the round of its barrier
            bool ok = true;
            while (ok) {
                ok = wait(item_full + 8 * item.at, item.turn, gave_up, a.status);
                const Item it = s_item[item.at];
                arrive(item_empty + 8 * item.at);
                item.go(1);
                if (!ok || it.steps < 0) break;
                if (it.steps == 0) continue;
                const int groups = it.end - it.begin > tokens ? 2 : 1;
                ok = wait(q_full + 8 * q.at, q.turn, gave_up, a.status);
                for (int j = 0; j < it.steps && ok; j++) {
                    ok = wait(full + 8 * kv.at, kv.turn, gave_up, a.status);
                    if (j >= it.dirty && ok) {
                        if (a.mask == nullptr) arrive(go);
                        ok = wait(clean + 8 * kv.at, clean_turns >> kv.at & 1, gave_up, a.status);
                        clean_turns ^= 1u << kv.at;
                    }
                    for (int g = 0; g < groups && ok; g++) {
                        if (scored >= B) ok = wait(used + 8 * buffer.at, buffer.turn ^ 1, gave_up, a.status);
                        after_sync();
                        if (!ok) break;
                        product_along<CHUNKS, kMmaRows * kTile, N * kTile>(tmem + N * buffer.at, s_q + q.at * F::kQueryBytes + g * F::kHalfBytes,
                                                                           s_k + kv.at * F::kTileBytes, depth, shape_s);
                        arrive_when_done(s_full + 8 * buffer.at);
                        scored = min(scored + 1, B);
                        buffer.go(1);
                    }
                    kv.go(1);
                }
                if (ok) arrive_when_done(q_empty + 8 * q.at);
                q.go(1);
            }
            arrive_when_done(scores_done);  // no product is under way when the tensor memory is freed
            drain(scores_done, 0);
        }
        __syncwarp();
    } else if (warp == 18) {
        if (elect()) {
            const unsigned shape_o = shape<T>((a.dim + 15) / 16 * 16, true);
            Ring<F::kItems> item;
            Ring<F::kStages> kv;
            Ring<B> buffer;
            unsigned o_turn[2] = {1, 1};  // of the halves' sums, which are free at first
            bool ok = true, o_used[2] = {false, false};
            while (ok) {
                ok = wait(item_full + 8 * item.at, item.turn, gave_up, a.status);
                const Item it = s_item[item.at];
                arrive(item_empty + 8 * item.at);
                item.go(1);
                if (!ok || it.steps < 0) break;
                const int groups = it.end - it.begin > tokens ? 2 : 1;
                for (int j = 0; j < it.steps && ok; j++) {
                    for (int i = 0; i < groups && ok; i++) {
                        const int g = alternate ? j & 1 : i;
                        const bool begins = j < (alternate ? 2 : 1);
                        ok = wait(p_full + 8 * buffer.at, buffer.turn, gave_up, a.status);
                        if (begins && ok) {  // the results of the tile before have been read
                            if (o_used[g]) ok = wait(o_empty + 8 * g, o_turn[g], gave_up, a.status);
                            o_used[g] = true;
                            o_turn[g] ^= 1;
                        }
                        after_sync();
                        if (!ok) break;
                        product_over<N / 16, N * kTile>(tmem + F::kOut + 64 * CHUNKS * g, tmem + N * buffer.at, s_v + kv.at * F::kTileBytes, shape_o, !begins);
                        arrive_when_done(used + 8 * buffer.at);
                        arrive_when_done(o_full + 8 * g);
                        buffer.go(1);
                    }
                    if (ok) arrive_when_done(empty + 8 * kv.at);
                    kv.go(1);
                }
            }
            arrive_when_done(sums_done);
            drain(sums_done, 0);
        }
        __syncwarp();
    } else if (warp == 19) {
        // Masked keys may be in any step, and are cleared as the copies come in.  Else it is the event's last step alone, for which
        // the scores ask: a warp that followed every step would cost the others 5 %.
        Ring<F::kItems> item;
        Ring<F::kStages> kv;
        unsigned go_turn = 0;
        bool ok = true;
        while (ok) {
            ok = wait_warp<true>(item_full + 8 * item.at, item.turn, gave_up, a.status);
            const Item it = s_item[item.at];
            __syncwarp();
            if (lane == 0) arrive(item_empty + 8 * item.at);
            item.go(1);
            if (!ok || it.steps < 0) break;
            for (int j = 0; j < it.steps && ok; j++, kv.go(1)) {
                if (j < it.dirty) continue;
                const int k0 = it.first + j * N;
                unsigned seen[W];
                const bool all = seen_words<W>(seen, a.mask, k0, it.keys_end - k0);
                if (a.mask != nullptr) {
                    ok = wait_warp<true>(full + 8 * kv.at, kv.turn, gave_up, a.status);
                } else {
                    ok = wait_warp<true>(go, go_turn, gave_up, a.status);
                    go_turn ^= 1;
                }
                if (!ok) break;
                if (!all) {
                    clear_unseen<W>(s_k + kv.at * F::kTileBytes, CHUNKS, seen);
                    clear_unseen<W>(s_v + kv.at * F::kTileBytes, CHUNKS, seen);
                    writes_before_products();
                }
                unsigned any = 0;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    s_bias[kv.at * N + 32 * w + lane] = (seen[w] >> lane) & 1u ? 0.f : -INFINITY;
                    any |= seen[w];
                }
                if (lane == 0) s_any[kv.at] = any != 0;
                __syncwarp();
                if (lane == 0) arrive(clean + 8 * kv.at);
            }
        }
    } else {
        const int g = warp >> 3, half = (warp >> 2) & 1, r = t & 127;  // the lane has row r of half tile g, and half of its columns
        const unsigned lanes = tmem + ((unsigned)(warp & 3) << 21), out = lanes + F::kOut + 64 * CHUNKS * g;
        float *maxima = reinterpret_cast<float *>(s_raw + F::kTiles + F::kMaxAt) + g * 3 * 2 * kMmaRows;  // [two in turn, and the sums][halves][rows]
        const unsigned meeting = meet + 8 * (g * 4 + (warp & 3));  // of the two warps that share rows
        unsigned meet_turn = 0;
        bool ok = true;
        const auto exchange = [&](float *both_halves, float mine) {
            both_halves[half * kMmaRows + r] = mine;
            __syncwarp();
            if (lane == 0) arrive(meeting);
            ok = wait_warp<true>(meeting, meet_turn, gave_up, a.status) && ok;
            meet_turn ^= 1;
            return both_halves[(half ^ 1) * kMmaRows + r];
        };
        constexpr int V = W / 2;
        const float c = a.scale * kLog2e;
        const pair c2 = pair_of(c, c);
        Ring<F::kItems> item;
        Ring<F::kStages> kv;
        Ring<B> buffer;
        unsigned o_turn = 0, clean_turns = 0;
        while (ok) {
            ok = wait_warp<true>(item_full + 8 * item.at, item.turn, gave_up, a.status);
            const Item it = s_item[item.at];
            if (!ok || it.steps < 0) break;
            const int groups = it.end - it.begin > tokens ? 2 : 1, begin = it.begin + (alternate ? 0 : g * tokens);
            // The second half may have no steps.  It must not go on all the same: a wait tells a barrier's phases apart by their parity only,
            // and would take the phase before the last for the next one.  It goes on when the first half has seen all scores of the item.
            if (g == 1 && it.steps > 0 && groups == 1 && (!alternate || it.steps == 1))
                ok = wait_warp<true>(item_done + 8 * item.at, item.turn, gave_up, a.status);
            __syncwarp();
            if (g == 1 && lane == 0) arrive(item_empty + 8 * item.at);
            const int n_rows = min(tokens, it.end - begin) * a.pack;
            const bool some = it.steps > (alternate ? g : 0);  // steps for this half
            int count = 0;
            const bool idle = (warp & 3) * 32 >= n_rows, store = r < n_rows;  // idle: none of the warp's rows counts
            float top = -INFINITY, sum = 0.f;
            bool any = false;  // whether a key is seen
            if (groups == 2 && g == 1 && it.steps > 0) buffer.go(1);  // this half's place among the two
            for (int j = 0; j < it.steps; j++, kv.go(1)) {
                const bool whole_step = j < it.dirty;
                const unsigned clean_turn = clean_turns >> kv.at & 1;
                if (!whole_step) clean_turns ^= 1u << kv.at;
                if (alternate ? (j & 1) != g : g >= groups) {  // the other half's buffers
                    buffer.go(1);
                    continue;
                }
                const unsigned rows = lanes + N * buffer.at + half * (N / 2);
                ok = wait_warp<true>(s_full + 8 * buffer.at, buffer.turn, gave_up, a.status) && ok;
                if (!whole_step) ok = wait_warp<true>(clean + 8 * kv.at, clean_turn, gave_up, a.status) && ok;
                any = any || whole_step || s_any[kv.at] != 0;
                // every phase of the sums' barrier is waited for: here, where they are scaled, else when this step's weights are done
                bool summed = count == 0;
                if (!idle) {
                    after_sync();
                    // The scores are read twice, 32 at a time: once for the maximum and once for the weights.  The loops stay loops: unrolled
                    // and in a second form for masked keys they were more instructions than the caches hold.
                    unsigned s[32];
                    const float *bias = s_bias + kv.at * N + half * (N / 2);
                    const auto read = [&](int w) {
                        tmem_load32(s, rows + 32 * w);
                        if (whole_step) return;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 add = *reinterpret_cast<const float4 *>(bias + 32 * w + i);
                            s[i] = __float_as_uint(__uint_as_float(s[i]) + add.x);
                            s[i + 1] = __float_as_uint(__uint_as_float(s[i + 1]) + add.y);
                            s[i + 2] = __float_as_uint(__uint_as_float(s[i + 2]) + add.z);
                            s[i + 3] = __float_as_uint(__uint_as_float(s[i + 3]) + add.w);
                        }
                    };
                    float m[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int w = 0; w < V; w++) {
                        read(w);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) m[(i >> 1) & 3] = max3(m[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                    }
                    float next = max2(max3(m[0], m[1], m[2]), m[3]);
                    next = max2(next, exchange(maxima + (count & 1) * 2 * kMmaRows, next));
                    // The sums are scaled again only where a row's maximum has grown by more than that.  The others of the warp stay as
                    // they are then, so that no result depends on which rows share a warp; and rows that do not count have no say: what
                    // stands there may differ from run to run.
                    const bool grown = store && ((next - top) * c > Weights<T>::kGrowth || next != next);
                    const float before = top;
                    if (count == 0 || grown) top = next;
                    if (count == 0) {
                    } else if (__any_sync(0xffffffffu, grown)) {
                        ok = wait_warp<true>(o_full + 8 * g, o_turn ^ 1, gave_up, a.status) && ok;
                        summed = true;
                        after_sync();
                        const float shrink = exp2_fast((before - (top == -INFINITY ? 0.f : top)) * c);
                        sum *= shrink;
                        for (int d = 16 * half; d < a.dim; d += 32) {
                            unsigned o[16];
                            tmem_load16(o, out + d);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                            tmem_store16(out + d, o);
                        }
                    }
                    const float base = (top == -INFINITY ? 0.f : top) * c - Weights<T>::kShift;
                    const pair base2 = pair_of(-base, -base);
                    pair sums[2] = {0, 0};
                    // The special function unit takes 8 cycles for a warp's exponentials; a quarter of them goes without it.  (There, a masked
                    // key gets 2^-126: its row of values is zero, and a sum of nothing else is told by its maximum.)
#pragma unroll 1
                    for (int w = 0; w < V; w++) {
                        if (V > 1) read(w);
                        unsigned p[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 x = parts(fma2(pair_of(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, base2));
                            const float2 e = i % 4 == 3 ? exp2_arithmetic(x) : make_float2(exp2_fast(x.x), exp2_fast(x.y));
                            sums[i & 1] = add2(sums[i & 1], pair_of(e.x, e.y));
                            p[i] = pack2<T>(e.x, e.y);
                        }
                        tmem_store16(rows + 16 * w, p);
                    }
                    const float2 both = parts(add2(sums[0], sums[1]));
                    sum += both.x + both.y;
                    tmem_stored();
                }
                if (!summed) ok = wait_warp<true>(o_full + 8 * g, o_turn ^ 1, gave_up, a.status) && ok;
                o_turn ^= 1;
                before_sync();
                __syncwarp();
                if (lane == 0) arrive(p_full + 8 * buffer.at);
                buffer.go(groups == 1 || (g == 1 && j == it.steps - 1) ? 1 : 2);
                count++;
            }
            if (g == 0) {  // in this order: the next item in this slot has the next phase
                __syncwarp();
                if (lane == 0) {
                    arrive(item_done + 8 * item.at);
                    arrive(item_empty + 8 * item.at);
                }
            }
            item.go(1);
            if (g >= groups && !alternate) continue;
            const bool done = some && ok && wait_warp<true>(o_full + 8 * g, o_turn ^ 1, gave_up, a.status);
            if (done) after_sync();
            const long long row = (long long)(begin + r / a.pack) * a.heads + it.head0 + r % a.pack;
            if (some && !idle) sum += exchange(maxima + 2 * 2 * kMmaRows, sum);
            // Scores of a query of NaN or infinity are no numbers where keys are cleared either, so that its maximum says nothing.
            const bool none = !any || top == -INFINITY;
            const float inv = none ? 0.f : 1.f / sum;
            const long long all_rows = (long long)a.n_q * a.heads;
            const bool parts = a.splits > 1 || alternate;
            const int part = alternate ? 2 * it.split + g : it.split;
            if (store && half == 0) {
                float *lse = parts ? a.part_lse + part * all_rows : a.lse;
                lse[row] = none ? -INFINITY : top * a.scale + (logf(sum) - Weights<T>::kShift * kLn2);
            }
            float *to_part = parts ? a.part + part * all_rows * a.dim : nullptr;
            if (!idle && (done || !parts)) {  // a part without keys has no weight
                const Rows to(row * a.dim, store);
                for (int d = 16 * half; d < a.dim; d += 32) {
                    unsigned o[16] = {};
                    if (done) {
                        tmem_load16(o, out + d);
                        if (none)
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = 0;
                    }
                    store16<T>(a.to, REST ? a.rest : nullptr, to_part, to, d, a.dim, o, inv);
                }
            }
            if (some) {
                before_sync();
                __syncwarp();
                if (lane == 0) arrive(o_empty + 8 * g);
            }
        }
    }
    before_sync();
    __syncthreads();
    after_sync();
    if (warp == 19) tmem_free(tmem, F::kColumns);
}

// ------------------------------------------------------------------------------------------------------------ backward
// Half precision reaches down to 2^-24 only, and a weight among many keys lies below that: weights are held 2^14 times as large
// there, and their gradients are scaled by a power of two under which none can overflow (|do.v - delta| <= 2 max|do| max|v|): one for
// each row of the gradient of queries, and, as the gradient of a key is a sum over the queries, one for each event there.
// Both factors are taken out of the float32 sums.
template <typename T> struct Range { static constexpr float kShift = 0.f; };
template <> struct Range<__half> { static constexpr float kShift = kHalfShift; };

// `row`: of the gradient, or -1 for the largest of the event
template <typename T> __device__ __forceinline__ float slope_factor(const Args &a, int event, long long row)
{
    if (Range<T>::kShift == 0.f || event >= a.n_events) return 1.f;
    const float bound = sqrtf(fresh(row < 0 ? a.bounds + 2 * event : a.norms + row)) * sqrtf(fresh(a.bounds + 2 * event + 1));
    return bound > 0.f && bound < 1e30f ? exp2f(-ceilf(log2f(bound))) : 1.f;
}

// Rows [from, to) of a tile as zeros; a whole warp.
__device__ __forceinline__ void clear_rows(unsigned tile, int chunks, int tile_rows, int from, int to)
{
    for (int c = 0; c < chunks; c++)
        for (int i = from * 8 + lane_id(); i < to * 8; i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(tile + c * tile_rows * kTile + i * 16), "r"(0) : "memory");
}

// Both gradients are the same walk.  A block keeps 128 rows of two tensors (KEYS: keys and values, else queries and grad) and the
// rows of the two others of the event pass by, 64 a step:
//   KEYS: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q;  else S = Q K^T, dP = dO V^T, dQ += dS K
// with a kept row per lane.  P and dS (16 bits) take the places of S and dP in tensor memory, from where they are an operand of the
// sums.  One block has a multiprocessor and all 512 columns: the sums, and as many buffers for S and dP as there is room for, so
// that two groups of four warps, which take the steps in turn, find the next step's scores done.  What bounds a step is how fast
// products can be issued (about 36 cycles each, 12 or 16 a step) and the exponentials (512 cycles), so scores and sums are issued by a
// thread each, that does nothing else, and rows that must not be summed over are cleared by a warp of their own.
// (Two blocks of 256 columns, each with one buffer, waited for products two thirds of the time: 16k x 16k rows, 8 heads of 64, 3.2 ms.)
template <int CHUNKS, bool KEYS> struct Grad {
    static constexpr int kStep = kMmaGradStep, kStages = CHUNKS == 1 ? 6 : 4, kThreads = 384;
    static constexpr int kTileBytes = kStep * kTile * CHUNKS, kKeptBytes = kMmaRows * kTile * CHUNKS;
    static constexpr int kBuffers = KEYS && CHUNKS == 2 ? 2 : 3, kSums = 128 * kBuffers, kSums2 = kSums + 64 * CHUNKS, kColumns = 512;
    static constexpr int kTiles = 2 * kKeptBytes + 2 * kStages * kTileBytes, kStats = 8 * 2 * kStep * 4, kSmem = kTiles + kStats + 512;
    static constexpr int kBarriers = 4 + 3 * kStages + 3 * kBuffers;
    static_assert((KEYS ? kSums2 : kSums) + 64 * CHUNKS <= kColumns && 8 * kBarriers + 8 <= 512, "room");
};

template <typename T, int CHUNKS, bool KEYS>
__global__ void __launch_bounds__(Grad<CHUNKS, KEYS>::kThreads, 1)
grad_mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps)
{
    pdl_begin();
    using F = Grad<CHUNKS, KEYS>;
    constexpr int N = F::kStep, W = N / 32, B = F::kBuffers;
    constexpr bool kScaled = Range<T>::kShift != 0.f;
    extern __shared__ __align__(1024) char s_raw[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int tokens = (KEYS ? N : kMmaRows) / a.pack;  // of a tile of queries
    const int kv = KEYS ? blockIdx.y : blockIdx.y * a.pack / a.group, packs = KEYS ? a.group / a.pack : 1;
    const Tile tile = KEYS ? find_tile(a.rs_k, a.n_k, a.n_events, kMmaRows, blockIdx.x) : find_tile(a.rs_q, a.n_q, a.n_events, tokens, blockIdx.x);
    if (tile.begin >= tile.end) return;
    const int n_rows = KEYS ? tile.end - tile.begin : (tile.end - tile.begin) * a.pack;
    const bool varies = tile.event < a.n_events && fresh(a.visible + tile.event) > 1;
    int2 others = KEYS ? rows_of(a.rs_q, a.n_q, a.n_events, tile.event) : rows_of(a.rs_k, a.n_k, a.n_events, tile.event);
    if (!KEYS && !varies) others.y = others.x;
    const int rows_a_step = KEYS ? tokens : N;
    const int2 part = part_of(max(0, (others.y - others.x + rows_a_step - 1) / rows_a_step), blockIdx.z, a.splits);
    const int steps = (part.y - part.x) * packs, first_row = others.x + part.x * rows_a_step;
    // Steps from this one on hold rows that must not be summed over: of another event, or keys that are masked.
    const int whole = (others.y - others.x) / rows_a_step;  // steps, of one head
    const int dirty = !KEYS && a.mask != nullptr ? 0 : max(0, (min(part.y, max(whole, part.x)) - part.x) * packs);

    const unsigned s_kept = smem_address(s_raw), s_kept2 = s_kept + F::kKeptBytes, s_step = s_kept2 + F::kKeptBytes,
                   s_step2 = s_step + F::kStages * F::kTileBytes;
    const unsigned bar = s_kept + F::kTiles + F::kStats, kept_full = bar, scores_done = bar + 8, all_done = scores_done + 8, go = all_done + 8, full = go + 8,
                   empty = full + 8 * F::kStages, clean = empty + 8 * F::kStages, s_full = clean + 8 * F::kStages, p_full = s_full + 8 * B, used = p_full + 8 * B;
    unsigned *s_tmem = reinterpret_cast<unsigned *>(s_raw + F::kTiles + F::kStats + 8 * F::kBarriers);
    volatile int *gave_up = reinterpret_cast<volatile int *>(s_tmem + 1);
    if (steps > 0) {
        if (t == 0) {
            for (int i = 0; i < F::kBarriers; i++) {
                const unsigned at = bar + 8 * i;
                barrier_init(at, at >= p_full && at < used ? 4 : at == kept_full ? 2 : 1);
            }
            barrier_init_done();
            *gave_up = 0;
        }
        if (warp == 11) tmem_alloc(s_tmem, F::kColumns);
        before_sync();
        __syncthreads();
        after_sync();
    }
    const unsigned tmem = steps > 0 ? *s_tmem : 0;

    if (warp == 8) {
        if (steps > 0 && elect()) {
            const int kept_head = KEYS ? kv : blockIdx.y * a.pack;
            arrive_expect(kept_full, KEYS ? 2 * F::kKeptBytes : 2 * CHUNKS * kTile * a.pack * tokens);
            for (int c = 0; c < CHUNKS; c++) {
                copy_box(s_kept + c * kMmaRows * kTile, KEYS ? &maps.k : &maps.q, kept_full, 64 * c, kept_head, tile.begin);
                copy_box(s_kept2 + c * kMmaRows * kTile, KEYS ? &maps.v : &maps.grad, kept_full, 64 * c, kept_head, tile.begin);
            }
            int copies = 0, row = first_row, p = 0;
            for (int j = 0; j < steps; j++) {
                const int stage = j % F::kStages, head = KEYS ? kv * a.group + p * a.pack : kv;
                if (j >= F::kStages && !wait(empty + 8 * stage, (j / F::kStages & 1) ^ 1, gave_up, a.status)) break;
                arrive_expect(full + 8 * stage, KEYS ? 2 * CHUNKS * kTile * a.pack * tokens : 2 * F::kTileBytes);
                for (int c = 0; c < CHUNKS; c++) {
                    copy_box(s_step + stage * F::kTileBytes + c * N * kTile, KEYS ? &maps.q : &maps.k, full + 8 * stage, 64 * c, head, row);
                    copy_box(s_step2 + stage * F::kTileBytes + c * N * kTile, KEYS ? &maps.grad : &maps.v, full + 8 * stage, 64 * c, head, row);
                }
                copies++;
                if (++p == packs) {
                    p = 0;
                    row += rows_a_step;
                }
            }
            // no copy is under way when the block leaves
            drain(kept_full, 0);
            for (int j = max(0, copies - F::kStages); j < copies; j++) drain(full + 8 * (j % F::kStages), j / F::kStages & 1);
        }
        __syncwarp();
    } else if (warp == 9) {
        if (steps > 0 && elect()) {
            const int depth = (a.dim + 15) / 16;
            const unsigned shape_s = shape<T>(N, false);
            bool ok = wait(kept_full, 0, gave_up, a.status);
            int stage = 0, b = 0;
            unsigned turn = 0, turn_b = 1;  // of the stages; of the buffers, which are free at first
            for (int j = 0; j < steps && ok; j++) {
                ok = wait(full + 8 * stage, turn, gave_up, a.status);
                if (KEYS && j >= dirty && ok) {
                    arrive(go);
                    ok = wait(clean + 8 * stage, (j - dirty) / F::kStages & 1, gave_up, a.status);
                }
                if (j >= B) ok = ok && wait(used + 8 * b, turn_b, gave_up, a.status);
                after_sync();
                if (ok) {
                    const unsigned to = tmem + 128 * b;
                    product_along<CHUNKS, kMmaRows * kTile, N * kTile>(to, s_kept, s_step + stage * F::kTileBytes, depth, shape_s);
                    product_along<CHUNKS, kMmaRows * kTile, N * kTile>(to + 64, s_kept2, s_step2 + stage * F::kTileBytes, depth, shape_s);
                    arrive_when_done(s_full + 8 * b);
                }
                if (++stage == F::kStages) stage = 0, turn ^= 1;
                if (++b == B) b = 0, turn_b ^= 1;
            }
            arrive_when_done(scores_done);  // no product is under way when the tensor memory is freed
            drain(scores_done, 0);
        }
        __syncwarp();
    } else if (warp == 10) {
        if (steps > 0 && elect()) {
            const unsigned shape_o = shape<T>((a.dim + 15) / 16 * 16, true);
            int stage = 0, b = 0;
            unsigned turn_b = 0;
            for (int j = 0; j < steps; j++) {
                if (!wait(p_full + 8 * b, turn_b, gave_up, a.status)) break;
                if (!KEYS && j >= dirty) {
                    if (a.mask == nullptr) arrive(go);
                    if (!wait(clean + 8 * stage, (j - dirty) / F::kStages & 1, gave_up, a.status)) break;
                }
                after_sync();
                const unsigned from = tmem + 128 * b;
                if (KEYS) product_over<N / 16, N * kTile>(tmem + F::kSums2, from, s_step2 + stage * F::kTileBytes, shape_o, j > 0);
                product_over<N / 16, N * kTile>(tmem + F::kSums, from + 64, s_step + stage * F::kTileBytes, shape_o, j > 0);
                arrive_when_done(used + 8 * b);
                arrive_when_done(empty + 8 * stage);
                if (++stage == F::kStages) stage = 0;
                if (++b == B) b = 0, turn_b ^= 1;
            }
            arrive_when_done(all_done);
            drain(all_done, 0);
        }
        __syncwarp();
    } else if (warp == 11) {
        if (KEYS && steps > 0 && a.pack * tokens < N) {  // rows that no copy writes
            for (int i = 0; i < F::kStages; i++) {
                clear_rows(s_step + i * F::kTileBytes, CHUNKS, N, a.pack * tokens, N);
                clear_rows(s_step2 + i * F::kTileBytes, CHUNKS, N, a.pack * tokens, N);
            }
        }
        writes_before_products();
        __syncwarp();
        if (lane == 0 && steps > 0) arrive(kept_full);
        for (int j = dirty; j < steps; j++) {
            const int stage = j % F::kStages, row = first_row + j / packs * rows_a_step;
            const unsigned step = s_step + stage * F::kTileBytes, step2 = s_step2 + stage * F::kTileBytes;
            unsigned seen[W];
            const bool all = KEYS || seen_words<W>(seen, a.mask, row, others.y - row);
            if (!(!KEYS && a.mask != nullptr ? wait_warp(full + 8 * stage, j / F::kStages & 1, gave_up, a.status)
                                             : wait_warp(go, (j - dirty) & 1, gave_up, a.status)))
                break;
            if (KEYS) {
                clear_rows(step, CHUNKS, N, (others.y - row) * a.pack, a.pack * tokens);
                clear_rows(step2, CHUNKS, N, (others.y - row) * a.pack, a.pack * tokens);
            } else if (!all) {
                clear_unseen<W>(step, CHUNKS, seen);
            }
            writes_before_products();
            __syncwarp();
            if (lane == 0) arrive(clean + 8 * stage);
        }
    } else {
        const int g = warp >> 2, r = t & 127;  // the lane has row r in every other step, beginning with step g
        const unsigned lanes = tmem + ((unsigned)(warp & 3) << 21);
        const bool idle = (warp & 3) * 32 >= n_rows, store = r < n_rows;
        // KEYS: of the columns, in the warp's own shared memory, negative, first the exponents' and then the slopes'.  Else of this
        // lane's row.
        float *stats = reinterpret_cast<float *>(s_raw + F::kTiles) + warp * 2 * N;
        const long long row = KEYS ? ((long long)(tile.begin + r) * a.kv_heads + kv)
                                   : (long long)(tile.begin + r / a.pack) * a.heads + blockIdx.y * a.pack + r % a.pack;
        const float scale = a.scale * kLog2e, factor = KEYS || store ? slope_factor<T>(a, tile.event, KEYS ? -1 : row) : 1.f;
        const pair c = pair_of(scale, scale), f = pair_of(factor, factor);
        pair shift = 0, delta = 0;
        unsigned seen_row = 0xffffffffu;
        if (KEYS) {
            seen_row = store && (a.mask == nullptr || fresh(a.mask + tile.begin + r) != 0) ? 0xffffffffu : 0u;
        } else {
            const float2 stat = store ? a.stats[row] : make_float2(INFINITY, 0.f);
            shift = pair_of(-stat.x, -stat.x);
            delta = pair_of(-stat.y * factor, -stat.y * factor);
        }
        // KEYS: the lane asks for two columns of the next step
        int token[2], head[2], p_next = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            token[w] = first_row + (KEYS ? (32 * w + lane) / a.pack : 0);
            head[w] = KEYS ? kv * a.group + (32 * w + lane) % a.pack : 0;
        }
        float2 mine[W];
        const auto next_stats = [&](int ahead) {
            for (p_next += ahead; p_next >= packs; p_next -= packs) {
                token[0] += rows_a_step;
                token[1] += rows_a_step;
            }
#pragma unroll
            for (int w = 0; w < W; w++)
                mine[w] = 32 * w + lane < a.pack * tokens && token[w] < others.y
                    ? a.stats[(long long)token[w] * a.heads + head[w] + p_next * a.pack] : make_float2(INFINITY, 0.f);
        };
        if (KEYS && g < steps) next_stats(g);
        int b = g, row_k = first_row + g * N;
        unsigned turn = 0;
        for (int j = g; j < steps; j += 2) {
            const unsigned rows = lanes + 128 * b;
            unsigned seen[W];
            bool all = true;
            if (KEYS) {
                __syncwarp();
#pragma unroll
                for (int w = 0; w < W; w++) {
                    stats[32 * w + lane] = -mine[w].x;
                    stats[N + 32 * w + lane] = -mine[w].y * factor;
                }
                if (j + 2 < steps) next_stats(2);
                __syncwarp();
            } else if (j >= dirty) {
                all = seen_words<W>(seen, a.mask, row_k, others.y - row_k);
            }
            row_k += 2 * N;
            if (wait_warp(s_full + 8 * b, turn, gave_up, a.status) && !idle) {
                after_sync();
#pragma unroll
                for (int w = 0; w < W; w++) {
                    unsigned s[32], d[32], p[16], q[16];
                    tmem_load32(s, rows + 32 * w, d, rows + 64 + 32 * w);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        pair x[2] = {shift, shift}, y[2] = {delta, delta};
                        if (KEYS) {
                            const ulonglong2 sx = *reinterpret_cast<const ulonglong2 *>(stats + 32 * w + i);
                            const ulonglong2 sy = *reinterpret_cast<const ulonglong2 *>(stats + N + 32 * w + i);
                            x[0] = sx.x; x[1] = sx.y; y[0] = sy.x; y[1] = sy.y;
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int at = i + 2 * h;
                            const float2 e = parts(fma2(pair_of(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), c, x[h]));
                            const float2 w2 = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                            const pair dp = pair_of(__uint_as_float(d[at]), __uint_as_float(d[at + 1]));
                            const float2 slope = parts(mul2(pair_of(w2.x, w2.y), kScaled ? fma2(dp, f, y[h]) : add2(dp, y[h])));
                            if (KEYS) {
                                p[at / 2] = pack2<T>(w2.x, w2.y) & seen_row;
                                q[at / 2] = pack2<T>(slope.x, slope.y) & seen_row;
                            } else {
                                q[at / 2] = pack2<T>(slope.x, slope.y);
                            }
                        }
                    }
                    if (!KEYS && !all) {
                        const unsigned word = w ? seen[1] : seen[0];
#pragma unroll
                        for (int i = 0; i < 16; i++) q[i] &= ((word >> (2 * i)) & 1u ? 0x0000ffffu : 0u) | ((word >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
                    }
                    // in place: this lane has read these columns
                    if (KEYS) tmem_store16(rows + 32 * w, p);
                    tmem_store16(rows + 64 + 32 * w, q);
                }
                tmem_stored();
            }
            before_sync();
            __syncwarp();
            if (lane == 0) arrive(p_full + 8 * b);
            b += 2;
            if (b >= B) b -= B, turn ^= 1;
        }
        const bool done = steps > 0 && wait_warp(all_done, 0, gave_up, a.status);
        if (done) after_sync();
        const float back = exp2f(-Range<T>::kShift);
        const long long all_rows = KEYS ? (long long)a.n_k * a.kv_heads : (long long)a.n_q * a.heads;
        // KEYS: the first group writes dv and the second dk; else they share the columns
        float *to_part = a.splits > 1 ? (KEYS && g == 0 ? a.part2 : a.part) + blockIdx.z * all_rows * a.dim : nullptr;
        void *to = KEYS && g == 0 ? a.to2 : a.to;
        const float by = KEYS && g == 0 ? back : a.scale * back / factor;
        const bool some = done && (varies || (KEYS && g == 0));
        const Rows place(row * a.dim, store);
        for (int d = KEYS ? 0 : 16 * g; d < a.dim; d += KEYS ? 16 : 32) {
            unsigned o[16] = {};
            if (some) {
                tmem_load16(o, lanes + (KEYS && g == 0 ? F::kSums2 : F::kSums) + d);
                if (KEYS)  // a key that is not seen: a weight of zero does not make up for a query of NaN
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] &= seen_row;
            }
            store16<T>(to, nullptr, to_part, place, d, a.dim, o, some ? by : 0.f);
        }
    }
    if (steps > 0) {
        before_sync();
        __syncthreads();
        after_sync();
        if (warp == 11) tmem_free(tmem, F::kColumns);
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

template <typename K, typename... More>
int launch(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const Args &a, const Maps &maps, More... more)
{
    HGC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    HGC_CUDA_TRY(launch_pdl(kernel, grid, threads, smem, stream, a, maps, more...));
    HGC_LAUNCH_CHECK();
    return HGC_OK;
}

template <typename T, int CHUNKS, bool KEYS> int grad_mma(const Args &a, const Maps &maps, cudaStream_t stream)
{
    using F = Grad<CHUNKS, KEYS>;
    const long long tiles = KEYS ? tile_count(a.n_k, kMmaRows, a.n_events) : tile_count(a.n_q, kMmaRows / a.pack, a.n_events);
    return launch(grad_mma_kernel<T, CHUNKS, KEYS>, dim3((unsigned)tiles, KEYS ? a.kv_heads : a.heads / a.pack, a.splits), F::kThreads, F::kSmem, stream, a,
                  maps);
}

template <typename T, int CHUNKS> int forward_mma(const Args &a, const Maps &maps, cudaStream_t stream)
{
    const int rows = kMmaRows / a.pack * (a.alternate ? 1 : 2);
    const long long tiles = tile_count(a.n_q, rows, a.n_events), items = tiles * (a.heads / a.pack) * a.splits;
    if (items > kMaxCount) return HGC_ERR_UNSUPPORTED;
    const int blocks = items < sm_count() ? (int)items : sm_count();
    if (items > blocks) HGC_CUDA_TRY(cudaMemsetAsync(a.counter, 0, sizeof(int), stream));
    const bool rest = a.rest != nullptr && a.splits == 1 && !a.alternate;  // parts are rounded where they are joined
    return launch(rest ? forward_mma_kernel<T, CHUNKS, true> : forward_mma_kernel<T, CHUNKS, false>, blocks, Forward<CHUNKS>::kThreads,
                  Forward<CHUNKS>::kSmem, stream, a, maps, (int)tiles, (int)items, a.alternate);
}

}  // namespace

bool mma_takes(const Args &a, int dtype)
{
    const auto aligned = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    return (dtype == HGC_FLOAT16 || dtype == HGC_BFLOAT16) && a.dim % 8 == 0 && a.n_q > 0 && a.n_k > 0 && rows_fit(a.q) && rows_fit(a.k) && rows_fit(a.v) &&
           aligned(a.to) && aligned(a.to2) && aligned(a.rest) && aligned(a.grad);
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

template <bool KEYS> static int grad(const Args &a, int dtype, cudaStream_t stream)
{
    const Strided grad{a.grad, (long long)a.heads * a.dim, a.dim};
    const int rows_q = (KEYS ? kMmaGradStep : kMmaRows) / a.pack, rows_k = KEYS ? kMmaRows : kMmaGradStep;
    Maps maps;
    if (const int rc = map_of(&maps.q, a.q, dtype, a.dim, a.heads, a.n_q, a.pack, rows_q)) return rc;
    if (const int rc = map_of(&maps.grad, grad, dtype, a.dim, a.heads, a.n_q, a.pack, rows_q)) return rc;
    if (const int rc = map_of(&maps.k, a.k, dtype, a.dim, a.kv_heads, a.n_k, 1, rows_k)) return rc;
    if (const int rc = map_of(&maps.v, a.v, dtype, a.dim, a.kv_heads, a.n_k, 1, rows_k)) return rc;
    if (dtype == HGC_FLOAT16) return a.dim <= 64 ? grad_mma<__half, 1, KEYS>(a, maps, stream) : grad_mma<__half, 2, KEYS>(a, maps, stream);
    return a.dim <= 64 ? grad_mma<__nv_bfloat16, 1, KEYS>(a, maps, stream) : grad_mma<__nv_bfloat16, 2, KEYS>(a, maps, stream);
}
int mma_grad_queries(const Args &a, int dtype, cudaStream_t stream) { return grad<false>(a, dtype, stream); }
int mma_grad_keys(const Args &a, int dtype, cudaStream_t stream) { return grad<true>(a, dtype, stream); }

}  // namespace attn
}  // namespace hgc
