// kv_select.cu — the blocks of the 4-bit cache that a query reads, by an upper
// bound of the int8 query's product with each block's keys.
//
// Two launches, the second programmatic: scores of every (row, key/value head,
// block) by int8 matrix instructions (m16n8k32: 16 query columns x 8 blocks x
// 32 bytes), then a warp or a thread block per (row, head) finds the n_select-th
// largest score by bisection over the scores' ordered bits, its keys in
// registers.
#include "kv_async.cuh"

namespace gofann {
namespace {

constexpr int kScoreThreads = 256;
// The score of a block without a page: no number, as a product that overflows
// is -inf and its block may be one that is always kept.
constexpr float kNoPage = __builtin_nanf("");

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Blocks that row `i` of a sequence may read: 0 where its position is negative.
__device__ __forceinline__ int row_blocks(int len, int n, int i)
{
    const int pos = len - n + i;
    return pos < 0 ? 0 : pos / kKvPage + 1;
}

// Columns of a row: the group's query heads, padded to a power of two (or a
// multiple of 16), so that the 16 columns of a warp hold whole rows or part of
// one.
struct SelectShape {
    int group, cols_per_row;
    int columns;                  // columns of a warp: 8 or 16
    int rows;                     // rows of a warp
    uint32_t splits, split_tiles; // parts of a row's blocks, their 16-block tiles
    uint32_t stride;              // floats of a score row
};

// The bounds of two times 8 blocks as B fragments: lane t takes the 16-byte
// pieces t of each 64 bytes of blocks g and g + 8 (the order of the k axis is
// free as long as the queries follow it), so that a load fills two fragments.
template <int D>
struct BlockTile {
    static constexpr int kPieces = 2 * D / 64;
    uint4 piece[2][kPieces];
    float scale[2];  // of blocks g, g + 8; negative where there is no page
};
// Pages of a lane's two blocks; -1 = past the sequence or not a page.
__device__ __forceinline__ void tile_pages(const gofann_kv_cache& cache, const gofann_kv_batch& b, uint32_t seq, int len,
                                           int block, int (&page)[2])
{
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int at = block + 8 * r;
        page[r] = -1;
        if (at * kKvPage < len) {
            page[r] = __ldg(b.page_table + static_cast<size_t>(seq) * b.max_pages + at);
            if (page[r] < 0 || static_cast<uint32_t>(page[r]) >= cache.n_pages) {
                page[r] = -1;
                kv_invalid(b);
            }
        }
    }
}
template <int D>
__device__ __forceinline__ void tile_bounds(const gofann_kv_cache& cache, uint32_t head, const int (&page)[2], BlockTile<D>& tile)
{
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const size_t entry = page[r] < 0 ? 0 : static_cast<size_t>(page[r]) * cache.n_kv_heads + head;
        const uint4* src = reinterpret_cast<const uint4*>(cache.bounds + entry * 2 * D) + t;
#pragma unroll
        for (int i = 0; i < BlockTile<D>::kPieces; ++i) {
            // (those of page 0 where there is none: the scale says so)
            const uint4 w = __ldg(src + 4 * i);
            tile.piece[r][i] = w;
        }
        const float scale = __ldg(cache.bound_scale + entry);
        tile.scale[r] = page[r] < 0 ? -1.0f : scale;
    }
}

// One query column in 8 bits as this lane's part of A fragments: dimensions
// 64 i + 16 t .. + 15, positive parts in the first pieces, negative ones in the
// others.  The four lanes of a column call it together; returns the scale, 0
// for a column that is zero or not finite.
template <int D, bool kBf16>
__device__ __forceinline__ float query_column(const gofann_kv_select_params& p, uint64_t at, bool on, bool wide,
                                              uint4 (&b)[2 * D / 64])
{
    uint4 raw[D / 32];
    float top = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint4& w = raw[2 * i + k];
            w = on ? load8(p.q, at + 64 * i + 8 * k, wide) : make_uint4(0u, 0u, 0u, 0u);
            float x[8];
            unpack8<kBf16>(w, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, fabsf(x[e]));
                nan |= x[e] != x[e];
            }
        }
    if (nan) top = __int_as_float(0x7f800000);  // fmaxf passes over it
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
    const bool fine = top > 0.0f && top < __int_as_float(0x7f800000);
    const float s = fine ? __fdiv_rn(top, 127.0f) : 0.0f, inv = fine ? __fdiv_rn(1.0f, s) : 0.0f;
    // rint of the quotients: by the reciprocal (off by less than 3e-5), unless
    // one is so near a half that the rounded quotient might fall to the other
    // side
    bool near = false;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        float x[8];
        unpack8<kBf16>(raw[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = x[e] * inv;
            near |= fabsf(t - rintf(t)) > 0.4999f;
        }
    }
    const auto split = [&](auto quotient) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            uint32_t up[4] = {0, 0, 0, 0}, down[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float x[8];
                unpack8<kBf16>(raw[2 * i + k], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int v = __float2int_rn(fminf(fmaxf(quotient(x[e]), -127.0f), 127.0f));
                    up[2 * k + e / 4] |= static_cast<uint32_t>(max(v, 0)) << (8 * (e & 3));
                    down[2 * k + e / 4] |= (static_cast<uint32_t>(min(v, 0)) & 0xffu) << (8 * (e & 3));
                }
            }
            b[i] = make_uint4(up[0], up[1], up[2], up[3]);
            b[D / 64 + i] = make_uint4(down[0], down[1], down[2], down[3]);
        }
    };
    if (near && fine)
        split([&](float x) { return __fdiv_rn(x, s); });
    else
        split([&](float x) { return fine ? x * inv : 0.0f; });
    return s;
}

// Scores of one warp: 16 query columns, kept as A fragments, against a part of
// the cache blocks, 16 at a time, the next ones' pages on their way.  kCols
// columns a row; 16 stands for rows of 16 columns and more (any multiple),
// which are done 16 at a time with the maximum so far in the score row.
// The maximum over a row's columns, which lanes 4 apart hold, is found by
// halves: at each step a lane keeps half of its values and sends the others.
// What bounds it: for a decode step the bounds' bytes (2 D + 4 a block) and how
// many of them are on their way (64 rows over 131072 tokens, 4 heads of 128:
// 104 MB in 31 us, 3.4 TB/s; fetching a tile ahead changes nothing), for a
// chunk the instructions around the products (16 products of 16 x 8 x 32 for
// 16 blocks at head_dim 128; 2043 rows over 40003 tokens, 2 heads: 52 us, 18 M
// instructions of a warp, 35 % of the issue slots).
// kGroups: 2, or 1 where a sequence's rows have 8 columns at most: the other
// half of the fragments is zero then and takes no registers (64 rows: 44 us
// against 47).
template <int D, bool kBf16, int kCols, int kGroups>
__global__ void __launch_bounds__(kScoreThreads, (D == 64 ? 3 : 2) + (kGroups == 1)) kv_score_kernel(gofann_kv_cache cache,
                                                                                  gofann_kv_batch batch,
                                                                                  gofann_kv_select_params p,
                                                                                  SelectShape sh, bool wide,
                                                                                  float* __restrict__ scores)
{
    constexpr int kPieces = BlockTile<D>::kPieces;
    constexpr int kOut = kCols == 1 ? kGroups : 1;  // rows that a lane writes
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    launch_next();
    // Few rows: a block's warps take the heads of a page, whose bounds lie side
    // by side in memory. Many: rows of one head, which share its bounds.
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kScoreThreads / 32) + (threadIdx.x >> 5);
    const uint64_t per_head = static_cast<uint64_t>(gridDim.x) * (kScoreThreads / 32) / cache.n_kv_heads;
    const uint64_t unit = kGroups == 2 ? item % per_head : item / cache.n_kv_heads;
    const uint32_t head = static_cast<uint32_t>(kGroups == 2 ? item / per_head : item - unit * cache.n_kv_heads);
    if (head >= cache.n_kv_heads) return;
    uint32_t seq, tile;
    const auto tiles = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>((n + sh.rows - 1) / sh.rows);
    };
    if (!kv_find<uint32_t>(batch.n_seqs, static_cast<uint32_t>(unit / sh.splits), tiles, seq, tile)) return;
    int first, n;
    kv_rows(batch, seq, first, n);
    const int len = kv_len(batch, seq);
    const int r0 = static_cast<int>(tile) * sh.rows, r1 = min(r0 + sh.rows, n);
    const int b0 = static_cast<int>(unit % sh.splits * sh.split_tiles) * 16;
    const int b1 = min(row_blocks(len, n, r1 - 1), b0 + static_cast<int>(sh.split_tiles) * 16);
    if (b0 >= b1) return;
    const int chunks = kCols == 16 ? sh.cols_per_row / 16 : 1;

    for (int chunk = 0; chunk < chunks; ++chunk) {
        int page[2];
        tile_pages(cache, batch, seq, len, b0 + g, page);
        // ---- the queries: columns g and g + 8
        uint32_t a[2 * kPieces][4] = {};
        float qs[kGroups];  // their scales; negative for a padding column
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            const int c = g + 8 * k;
            const int row = kCols == 16 ? r0 : r0 + c / kCols, h = kCols == 16 ? chunk * 16 + c : c % kCols;
            const bool on = row < r1 && h < sh.group;
            const uint64_t at = static_cast<uint64_t>(first + (on ? row : r0)) * p.q_stride +
                                static_cast<uint64_t>(head * sh.group + (on ? h : 0)) * D + 16 * t;
            uint4 q[kPieces];
            const float s = query_column<D, kBf16>(p, at, on, wide, q);
            qs[k] = on ? s : -1.0f;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                a[2 * i][k] = q[i].x, a[2 * i][2 + k] = q[i].y;
                a[2 * i + 1][k] = q[i].z, a[2 * i + 1][2 + k] = q[i].w;
            }
        }
        // ---- what this lane writes: of rows `mine`, blocks `off` (and off + 1)
        constexpr bool kTwo = kGroups == 2;
        int mine, off = 2 * t;
        if (kCols == 16) mine = 0, off += g >> 2;
        if (kCols == 8) mine = kTwo ? g >> 2 : 0, off += kTwo ? (g >> 1) & 1 : g >> 2;
        if (kCols == 4) mine = kTwo ? (g & 2) + (g >> 2) : g >> 2, off += kTwo ? g & 1 : (g >> 1) & 1;
        if (kCols == 2) mine = kTwo ? 4 * (g & 1) + (g >> 1) : g >> 1, off += kTwo ? 0 : g & 1;
        if (kCols == 1) mine = g;
        float* out[kOut];
        int blocks[kOut];
#pragma unroll
        for (int e = 0; e < kOut; ++e) {
            const int r = r0 + mine + 8 * e;
            blocks[e] = r < r1 ? row_blocks(len, n, r) : 0;
            out[e] = scores + (static_cast<size_t>(first + min(r, r1 - 1)) * cache.n_kv_heads + head) * sh.stride + off;
        }
        constexpr int kHeld = kCols == 16 ? 4 : kCols >= (kTwo ? 8 : 4) ? kCols / (kTwo ? 4 : 2) : 1;
        const bool writes = g % kHeld == 0;  // lanes that hold the same values
        for (int at = b0; at < b1; at += 16) {
            BlockTile<D> now;
            tile_bounds<D>(cache, head, page, now);
            if (at + 16 < b1) tile_pages(cache, batch, seq, len, at + 16 + g, page);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                int acc[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    mma_s8(acc, a[2 * i], now.piece[u][i].x, now.piece[u][i].y);
                    mma_s8(acc, a[2 * i + 1], now.piece[u][i].z, now.piece[u][i].w);
                }
                // acc: columns g, g + 8 x blocks 2t, 2t + 1 of the eight
                float v[kGroups][2];
#pragma unroll
                for (int k = 0; k < kGroups; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        v[k][e] = qs[k] < 0.0f ? kNegInf : __fmul_rn(static_cast<float>(acc[2 * k + e]), qs[k]);
                // halves that go: the other column group's, then the other block's
                const auto keep_group = [&](bool second, int lanes) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float got = __shfl_xor_sync(kFull, second ? v[0][e] : v[kGroups - 1][e], lanes);
                        v[0][e] = fmaxf(second ? v[kGroups - 1][e] : v[0][e], got);
                    }
                };
                const auto keep_block = [&](bool second, int lanes) {
                    const float got = __shfl_xor_sync(kFull, second ? v[0][0] : v[0][1], lanes);
                    v[0][0] = fmaxf(second ? v[0][1] : v[0][0], got);
                };
                const auto same = [&](int lanes) { v[0][0] = fmaxf(v[0][0], __shfl_xor_sync(kFull, v[0][0], lanes)); };
                if (kCols == 16) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[0][e] = fmaxf(v[0][e], v[kGroups - 1][e]);
                    keep_block(g & 4, 16), same(8), same(4);
                }
                if (kCols == 8 && kTwo) keep_group(g & 4, 16), keep_block(g & 2, 8), same(4);
                if (kCols == 8 && !kTwo) keep_block(g & 4, 16), same(8), same(4);
                if (kCols == 4 && kTwo) keep_group(g & 2, 8), keep_block(g & 1, 4);
                if (kCols == 4 && !kTwo) keep_block(g & 2, 8), same(4);
                if (kCols == 2 && kTwo) keep_group(g & 1, 4);
                if (kCols == 2 && !kTwo) keep_block(g & 1, 4);
                constexpr int kBlocks = kCols >= (kTwo ? 4 : 2) ? 1 : 2;  // blocks that a lane writes
#pragma unroll
                for (int w = 0; w < kBlocks; ++w) {
                    const float scale = __shfl_sync(kFull, now.scale[u], 4 * (off + w));
#pragma unroll
                    for (int e = 0; e < kOut; ++e) {
                        if (!writes || at + 8 * u + off + w >= blocks[e]) continue;
                        float* o = out[e] + at + 8 * u + w;
                        float x = v[e][w];
                        if (kCols == 16 && chunk > 0) x = fmaxf(x, *o);
                        if (chunk == chunks - 1) x = scale < 0.0f ? kNoPage : __fmul_rn(x, scale);
                        *o = x;
                    }
                }
            }
        }
    }
}

// Scores as unsigned keys of the same order; -0 counts as 0, forced blocks
// above everything, blocks without a page below everything.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kPickThreads = 256;

// The largest n_select of a row's scores, kWarps warps a row, up to kKeys keys
// a lane in registers (block kWarps 32 i + place): bisection, bit by bit from
// the top, for the largest key that at least n_select keys reach; all above it
// and the first ones at it are taken, in block order.  The scores come from L2:
// what bounds it is the chain of loads, up to 32 counts and the ranks (256 rows
// of 2048 blocks 15 us, 4086 rows of 626 blocks 26 us).
template <int kWarps, int kKeys>
__global__ void __launch_bounds__(kPickThreads) kv_pick_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                               gofann_kv_select_params p, uint32_t stride,
                                                               const float* __restrict__ scores)
{
    constexpr int kRows = kPickThreads / 32 / kWarps;  // rows of a thread block
    __shared__ uint32_t sums[2][8];
    if (blockIdx.x == 0) kv_check_sequences(batch, threadIdx.x, kPickThreads);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, place = threadIdx.x % (32 * kWarps);
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * kRows + warp / kWarps;
    if (item >= static_cast<uint64_t>(batch.n_rows) * cache.n_kv_heads) {  // whole warps (kWarps 8: whole blocks)
        wait_previous();
        return;
    }
    const uint32_t row = static_cast<uint32_t>(item / cache.n_kv_heads);
    uint32_t seq = 0, at = 0;
    const auto rows = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>(n);
    };
    int blocks = 0;
    if (kv_find<uint32_t>(batch.n_seqs, row, rows, seq, at)) {
        int first, n;
        kv_rows(batch, seq, first, n);
        blocks = row_blocks(kv_len(batch, seq), n, static_cast<int>(at));
    }
    wait_previous();
    const float* sc = scores + item * stride;
    int32_t* ids = p.ids + item * p.n_select;
    float* out = p.scores ? p.scores + item * p.n_select : nullptr;
    const uint32_t want = p.n_select;
    uint32_t key[kKeys];
    uint32_t valid = 0;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const int b = 32 * kWarps * i + place;
        key[i] = 0;
        if (b < blocks) {
            const float x = __ldcg(sc + b);
            if (x == x) {
                key[i] = b < static_cast<int>(p.n_first) || b >= blocks - static_cast<int>(p.n_recent) ? 0xffffffffu
                                                                                                        : order_key(x);
                ++valid;
            }
        }
    }
    int turn = 0;
    // the sum of a count over the row's warps, and over those before this one
    const auto row_sum = [&](uint32_t c, uint32_t& before) {
        if (kWarps == 1) {
            before = 0;
            return c;
        }
        turn ^= 1;
        if (lane == 0) sums[turn][warp] = c;
        __syncthreads();
        uint32_t all = 0;
        before = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t v = sums[turn][w];
            all += v;
            if (w < warp) before += v;
        }
        return all;
    };
    const auto row_max = [&](uint32_t c) {
        if (kWarps == 1) return c;
        turn ^= 1;
        if (lane == 0) sums[turn][warp] = c;
        __syncthreads();
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = max(m, sums[turn][w]);
        return m;
    };
    uint32_t before;
    const uint32_t present = row_sum(__reduce_add_sync(kFull, valid), before);
    uint32_t limit = 1, ties = 0xffffffffu;  // keys from `limit` on, of those at it the first `ties`
    if (present > want) {
        // the bits that all but the forced keys share need no bisection
        uint32_t most = 0, least = ~0u;
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
            if (key[i] != 0xffffffffu) most = max(most, key[i]);
            if (key[i] != 0) least = min(least, key[i]);
        }
        most = row_max(__reduce_max_sync(kFull, most));
        least = ~row_max(~__reduce_min_sync(kFull, least));
        const uint32_t differ = most ^ least;
        const int high = differ ? 31 - __clz(differ) : -1;
        limit = high < 31 ? least & ~((2u << (high < 0 ? 0 : high)) - 1u) : 0u;
        if (high < 0) limit = least;
        uint32_t above = present;  // keys that reach `limit`
        for (int bit = high; bit >= 0 && above != want; --bit) {
            const uint32_t try_at = limit | (1u << bit);
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) c += key[i] >= try_at;
            c = row_sum(__reduce_add_sync(kFull, c), before);
            if (c >= want) {
                limit = try_at;
                above = c;
            }
        }
        if (above != want) {
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) c += key[i] > limit;
            ties = want - row_sum(__reduce_add_sync(kFull, c), before);
        }
    }
    uint32_t taken = 0, tied = 0;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        if (32 * kWarps * i >= blocks) break;
        const bool tie = key[i] == limit, more = key[i] > limit;
        const unsigned tb = __ballot_sync(kFull, tie), ab = __ballot_sync(kFull, more);
        // counts of both, packed
        uint32_t earlier;
        const uint32_t all = row_sum(__popc(ab) | (__popc(tb) << 16), earlier);
        const unsigned below = (1u << lane) - 1u;
        const uint32_t a0 = taken + (earlier & 0xffff) + __popc(ab & below);
        const uint32_t t0 = tied + (earlier >> 16) + __popc(tb & below);
        if (more || (tie && t0 < ties)) {
            const uint32_t slot = a0 + (t0 < ties ? t0 : ties);
            const int b = 32 * kWarps * i + place;
            ids[slot] = b;
            if (out) out[slot] = __ldcg(sc + b);
        }
        taken += all & 0xffff;
        tied += all >> 16;
    }
    const uint32_t filled = taken + (tied < ties ? tied : ties);
    for (uint32_t i = filled + place; i < want; i += 32 * kWarps) {
        ids[i] = -1;
        if (out) out[i] = kNegInf;
    }
}

// The same for rows of any length, a thread block a row: the limit by four
// passes of a histogram over the scores in memory.
__global__ void __launch_bounds__(kPickThreads) kv_pick_long_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                    gofann_kv_select_params p, uint32_t stride,
                                                                    const float* __restrict__ scores)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t warp_sum[kPickThreads / 32][2];
    __shared__ uint32_t found_digit, found_rank;
    const uint32_t row = blockIdx.x, head = blockIdx.y;
    if (row == 0 && head == 0) kv_check_sequences(batch, threadIdx.x, kPickThreads);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t seq = 0, at = 0;
    const auto rows = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>(n);
    };
    int blocks = 0;
    if (kv_find<uint32_t>(batch.n_seqs, row, rows, seq, at)) {
        int first, n;
        kv_rows(batch, seq, first, n);
        blocks = row_blocks(kv_len(batch, seq), n, static_cast<int>(at));
    }
    wait_previous();
    const float* sc = scores + (static_cast<size_t>(row) * cache.n_kv_heads + head) * stride;
    int32_t* ids = p.ids + (static_cast<size_t>(row) * cache.n_kv_heads + head) * p.n_select;
    float* out = p.scores ? p.scores + (static_cast<size_t>(row) * cache.n_kv_heads + head) * p.n_select : nullptr;
    const int want = static_cast<int>(p.n_select);
    const auto key_of = [&](int b) {
        const float x = __ldcg(sc + b);
        if (x != x) return 0u;
        return b < static_cast<int>(p.n_first) || b >= blocks - static_cast<int>(p.n_recent) ? 0xffffffffu : order_key(x);
    };
    // the smallest key taken, and how many of its blocks (lowest first)
    uint32_t limit = 0, ties = 0xffffffffu;
    if (blocks > want) {
        uint32_t rank = static_cast<uint32_t>(want);  // the rank-th largest among keys that match `limit` so far
        for (int shift = 24; shift >= 0; shift -= 8) {
            hist[threadIdx.x] = 0;
            __syncthreads();
            for (int b = threadIdx.x; b < blocks; b += kPickThreads) {
                const uint32_t k = key_of(b);
                if (shift == 24 || (k >> (shift + 8)) == (limit >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (warp == 0) {
                // counts of digits from 255 down, eight per lane
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - (lane * 8 + i)];
                uint32_t before = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t v = __shfl_up_sync(kFull, before, off);
                    if (lane >= off) before += v;
                }
                before -= sum;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (before < rank && before + c[i] >= rank) {
                        found_digit = 255 - (lane * 8 + i);
                        found_rank = rank - before;
                    }
                    before += c[i];
                }
            }
            __syncthreads();
            limit |= found_digit << shift;
            rank = found_rank;
        }
        ties = rank;
    }
    // blocks above the limit and the first `ties` at it, in block order
    uint32_t taken = 0, tied = 0;
    for (int b0 = 0; b0 < blocks; b0 += kPickThreads) {
        const int b = b0 + threadIdx.x;
        const uint32_t k = b < blocks ? key_of(b) : 0u;
        const bool tie = b < blocks && k == limit && k != 0, above = b < blocks && k > limit;
        const unsigned tb = __ballot_sync(kFull, tie), ab = __ballot_sync(kFull, above);
        if (lane == 0) {
            warp_sum[warp][0] = __popc(ab);
            warp_sum[warp][1] = __popc(tb);
        }
        __syncthreads();
        uint32_t a0 = taken, t0 = tied;
#pragma unroll
        for (int w = 0; w < kPickThreads / 32; ++w) {
            if (w < warp) {
                a0 += warp_sum[w][0];
                t0 += warp_sum[w][1];
            }
            taken += warp_sum[w][0];
            tied += warp_sum[w][1];
        }
        const unsigned below = (1u << lane) - 1u;
        a0 += __popc(ab & below);
        t0 += __popc(tb & below);
        if (above || (tie && t0 < ties)) {
            const uint32_t slot = a0 + (t0 < ties ? t0 : ties);
            ids[slot] = b;
            if (out) out[slot] = __ldcg(sc + b);
        }
        __syncthreads();
    }
    const uint32_t filled = taken + (tied < ties ? tied : ties);
    for (uint32_t i = filled + threadIdx.x; i < static_cast<uint32_t>(want); i += kPickThreads) {
        ids[i] = -1;
        if (out) out[i] = kNegInf;
    }
}

// Row tiles of a call: a sequence of n rows has at most n / rows + 1, and at
// most n.
uint64_t row_tiles(const gofann_kv_batch& b, const SelectShape& s)
{
    const uint64_t bound = static_cast<uint64_t>(b.n_rows) / s.rows + b.n_seqs;
    return bound < b.n_rows ? bound : b.n_rows;
}

SelectShape select_shape(const gofann_kv_cache& c, const gofann_kv_batch& b, const gofann_kv_select_params& p)
{
    SelectShape s;
    s.group = static_cast<int>(p.n_heads / c.n_kv_heads);
    int cols = 1;
    while (cols < 8 && cols < s.group) cols *= 2;
    s.cols_per_row = s.group > 8 ? (s.group + 15) / 16 * 16 : cols;
    // columns of a warp: 8, if no sequence has more
    s.columns = s.cols_per_row <= 8 && static_cast<uint64_t>(b.max_rows) * s.cols_per_row <= 8 ? 8 : 16;
    s.rows = s.cols_per_row > 8 ? 1 : s.columns / s.cols_per_row;
    // Enough parts of a row's blocks for 16 (8 columns) or 12 warps an SM: each
    // part finds its sequence and rounds its queries anew. Both kernels at 64
    // rows over 131072 tokens: 8 an SM 55 us, 12 48 us, 16 44 us, 32 51 us; at
    // 2043 rows over 40003: 8 and 12 71 us, 16 74 us, 32 78 us.
    const uint32_t tiles = (b.max_pages + 15) / 16;
    const uint64_t units = row_tiles(b, s) * c.n_kv_heads, want = (s.columns == 8 ? 16ull : 12ull) * (sm_count() > 0 ? sm_count() : 1);
    uint64_t splits = units ? (want + units - 1) / units : 1;
    if (splits > tiles) splits = tiles;
    if (splits < 1) splits = 1;
    s.split_tiles = static_cast<uint32_t>((tiles + splits - 1) / splits);
    s.splits = s.split_tiles ? (tiles + s.split_tiles - 1) / s.split_tiles : 1;
    s.stride = (b.max_pages + 3) / 4 * 4;
    return s;
}

template <int D, bool kBf16>
void launch_score(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_select_params& p,
                  const SelectShape& s, bool wide, float* scores, dim3 grid, cudaStream_t cs)
{
    const auto go = [&](auto* kernel) { kernel<<<grid, kScoreThreads, 0, cs>>>(cache, batch, p, s, wide, scores); };
    const bool one = s.columns == 8;
    switch (s.cols_per_row) {
        case 1: return one ? go(kv_score_kernel<D, kBf16, 1, 1>) : go(kv_score_kernel<D, kBf16, 1, 2>);
        case 2: return one ? go(kv_score_kernel<D, kBf16, 2, 1>) : go(kv_score_kernel<D, kBf16, 2, 2>);
        case 4: return one ? go(kv_score_kernel<D, kBf16, 4, 1>) : go(kv_score_kernel<D, kBf16, 4, 2>);
        case 8: return one ? go(kv_score_kernel<D, kBf16, 8, 1>) : go(kv_score_kernel<D, kBf16, 8, 2>);
        default: return go(kv_score_kernel<D, kBf16, 16, 2>);
    }
}

}  // namespace
}  // namespace gofann

using namespace gofann;

extern "C" {

size_t gofann_kv_select_scratch_bytes(const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                                      const gofann_kv_select_params* params)
{
    if (!cache || !batch || !params || cache->n_kv_heads == 0 || params->n_heads < cache->n_kv_heads) return 0;
    const SelectShape s = select_shape(*cache, *batch, *params);
    return static_cast<size_t>(batch->n_rows) * cache->n_kv_heads * s.stride * sizeof(float);
}

int gofann_kv_select(const gofann_kv_cache* cache, const gofann_kv_batch* batch, const gofann_kv_select_params* params,
                     void* scratch, size_t scratch_bytes, void* stream)
{
    if (!params) return fail(GOFANN_ERR_INVALID, "kv_select: null descriptor");
    const gofann_kv_select_params& p = *params;
    int st = kv_check("kv_select", cache, batch, p.dtype, p.n_heads);
    if (st != GOFANN_OK) return st;
    const uint32_t d = cache->head_dim;
    if (p.n_select == 0 || p.n_select > GOFANN_KV_MAX_SELECT)
        return fail(GOFANN_ERR_UNSUPPORTED, "kv_select: n_select %u (1 .. %u)", p.n_select, GOFANN_KV_MAX_SELECT);
    if (p.n_first > p.n_select || p.n_recent > p.n_select - p.n_first)
        return fail(GOFANN_ERR_INVALID, "kv_select: n_first %u + n_recent %u above n_select %u", p.n_first, p.n_recent,
                    p.n_select);
    if (batch->n_rows == 0) return GOFANN_OK;
    if (!cache->bounds || !cache->bound_scale || !p.q || !p.ids)
        return fail(GOFANN_ERR_INVALID, "kv_select: null bounds, queries or ids");
    if ((reinterpret_cast<uintptr_t>(cache->bounds) & 15) || (reinterpret_cast<uintptr_t>(p.q) & 1))
        return fail(GOFANN_ERR_INVALID, "kv_select: bounds must be 16-byte, queries 2-byte aligned");
    if (p.q_stride < static_cast<uint64_t>(p.n_heads) * d)
        return fail(GOFANN_ERR_INVALID, "kv_select: a row stride is shorter than its row");
    if (batch->max_pages == 0 || cache->n_pages == 0) return fail(GOFANN_ERR_INVALID, "kv_select: rows without pages");
    const size_t need = gofann_kv_select_scratch_bytes(cache, batch, params);
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255))
        return fail(GOFANN_ERR_INVALID, "kv_select: scratch must be 256-byte aligned");
    if (scratch_bytes < need)
        return fail(GOFANN_ERR_CAPACITY, "kv_select: scratch of %zu bytes, %zu needed", scratch_bytes, need);
    const SelectShape s = select_shape(*cache, *batch, p);
    // whole blocks of each head's warps
    const uint64_t units = (row_tiles(*batch, s) * s.splits + kScoreThreads / 32 - 1) / (kScoreThreads / 32) * cache->n_kv_heads;
    const uint64_t items = static_cast<uint64_t>(batch->n_rows) * cache->n_kv_heads;
    if (units > 0x7fffffffull || items > 0x7fffffffull)
        return fail(GOFANN_ERR_UNSUPPORTED, "kv_select: %u rows of %u heads (2^31 - 1 at most)", batch->n_rows,
                    cache->n_kv_heads);
    float* scores = static_cast<float*>(scratch);
    cudaStream_t cs = as_stream(stream);
    const dim3 grid(static_cast<uint32_t>(units));
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && (p.q_stride & 7) == 0;
    if (d == 64)
        p.dtype == GOFANN_DTYPE_BF16 ? launch_score<64, true>(*cache, *batch, p, s, wide, scores, grid, cs)
                                     : launch_score<64, false>(*cache, *batch, p, s, wide, scores, grid, cs);
    else
        p.dtype == GOFANN_DTYPE_BF16 ? launch_score<128, true>(*cache, *batch, p, s, wide, scores, grid, cs)
                                     : launch_score<128, false>(*cache, *batch, p, s, wide, scores, grid, cs);
    GOFANN_CHECK_LAUNCH("kv_score_kernel");
    // A row's keys stay in registers up to 2048 blocks; a warp is enough for
    // 1024 where there are rows for every SM.  Both launches, us: 2043 rows x 2
    // heads of 626 blocks, a warp with 20 keys a lane 70, with 32 keys 84, eight
    // warps 88, keys in memory 83; 64 rows x 4 heads of 2048 blocks, eight warps
    // with 8 keys a lane 44, keys in memory 45; 4 rows x 4 heads of 2500
    // blocks, 64 keys a lane 23, keys in memory 16.
    const bool single = items >= 8ull * sm_count() && batch->max_pages <= 1024;
    const bool in_memory = batch->max_pages > 2048;
    const auto pick = in_memory ? kv_pick_long_kernel
                      : !single ? kv_pick_kernel<8, 8>
                      : batch->max_pages <= 256 ? kv_pick_kernel<1, 8>
                      : batch->max_pages <= 640 ? kv_pick_kernel<1, 20>
                                                : kv_pick_kernel<1, 32>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = in_memory ? dim3(batch->n_rows, cache->n_kv_heads)
                                           : dim3(static_cast<uint32_t>(single ? (items + 7) / 8 : items));
    cfg.blockDim = dim3(kPickThreads);
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, pick, *cache, *batch, p, s.stride, static_cast<const float*>(scores));
    if (e != cudaSuccess) return cuda_status(e, "kv_pick_kernel");
    return GOFANN_OK;
}

}  // extern "C"
