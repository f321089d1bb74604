// kv_select.cu — the blocks of the 4-bit cache that a query reads, by an int8
// upper bound of q.k over each block.
//
// Two launches: scores of every (row, key/value head, block) by int8 matrix
// instructions (m16n8k32: 16 blocks x 8 query columns x 32 bytes), then one
// block per (row, head) picks the n_select largest by a radix select over the
// scores' ordered bits.
#include "kv_common.cuh"

namespace gofann {
namespace {

constexpr int kScoreThreads = 256;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreBlocks = 16 * kScoreWarps;  // cache blocks of one thread block
constexpr int kScoreCols = 64;                  // query columns of one thread block

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
// multiple of 8), so that an 8-column tile holds whole rows or part of one.
struct SelectShape {
    int group, cols_per_row, rows_per_block;
    uint32_t block_tiles, stride;  // kScoreBlocks tiles of max_pages; floats of a score row
};

template <int D>
__global__ void __launch_bounds__(kScoreThreads) kv_score_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                 gofann_kv_select_params p, SelectShape sh,
                                                                 float* __restrict__ scores)
{
    extern __shared__ __align__(16) unsigned char smem[];
    int8_t* q8 = reinterpret_cast<int8_t*>(smem);               // [cols][2 D + 16]: positive parts, negative parts
    constexpr int kStride = 2 * D + 16;
    float* qs = reinterpret_cast<float*>(smem + static_cast<size_t>(sh.rows_per_block) * sh.cols_per_row * kStride);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t head = blockIdx.y;
    uint32_t seq, tile;
    const uint32_t row_tile = blockIdx.x / sh.block_tiles, block_tile = blockIdx.x % sh.block_tiles;
    const auto tiles = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>((n + sh.rows_per_block - 1) / sh.rows_per_block);
    };
    if (!kv_find(batch.n_seqs, row_tile, tiles, seq, tile)) return;
    int first, n;
    kv_rows(batch, seq, first, n);
    const int len = kv_len(batch, seq);
    const int r0 = static_cast<int>(tile) * sh.rows_per_block;
    const int r1 = r0 + sh.rows_per_block < n ? r0 + sh.rows_per_block : n;
    const int b0 = static_cast<int>(block_tile) * kScoreBlocks;
    if (b0 >= row_blocks(len, n, r1 - 1)) return;

    // ---- this warp's 16 blocks as A fragments: lane t takes the 16-byte
    // pieces t of each 64 bytes of rows g and g + 8 (the order of the k axis
    // is free as long as q8 follows it)
    constexpr int kPieces = 2 * D / 64;
    uint4 lo4[kPieces], hi4[kPieces];
    float scale[2];
    int page[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int b = b0 + warp * 16 + g + 8 * r;
        page[r] = -1;
        if (b * kKvPage < len) {
            page[r] = __ldg(batch.page_table + static_cast<size_t>(seq) * batch.max_pages + b);
            if (page[r] < 0 || static_cast<uint32_t>(page[r]) >= cache.n_pages) {
                page[r] = -1;
                kv_invalid(batch);
            }
        }
        const size_t entry = page[r] < 0 ? 0 : static_cast<size_t>(page[r]) * cache.n_kv_heads + head;
        const uint4* src = reinterpret_cast<const uint4*>(cache.bounds + entry * 2 * D) + t;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint4 w = page[r] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(src + 4 * i);
            if (r == 0) lo4[i] = w; else hi4[i] = w;
        }
        scale[r] = page[r] < 0 ? 0.0f : __ldg(cache.bound_scale + entry);
    }

    // ---- int8 queries of the rows, one warp per column
    const int cols = (r1 - r0) * sh.cols_per_row;
    for (int c = warp; c < (cols + 7) / 8 * 8; c += kScoreWarps) {
        const int r = c / sh.cols_per_row, h = c % sh.cols_per_row;
        float x[D / 32];
        const bool on = c < cols && h < sh.group;
        const uint64_t at = static_cast<uint64_t>(first + r0 + r) * p.q_stride + (head * sh.group + h) * D;
        float a = 0.0f;
        bool fine = true;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = on ? kv_load(p.q, at + lane + 32 * i, p.dtype) : 0.0f;
            fine &= fabsf(x[i]) < __int_as_float(0x7f800000);
            a = fmaxf(a, fabsf(x[i]));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(kFull, a, off));
        fine = __all_sync(kFull, fine) && a > 0.0f;
        const float s = fine ? __fdiv_rn(a, 127.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int v = fine ? static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.0f), 127.0f)) : 0;
            q8[c * kStride + lane + 32 * i] = static_cast<int8_t>(v > 0 ? v : 0);
            q8[c * kStride + D + lane + 32 * i] = static_cast<int8_t>(v < 0 ? v : 0);
        }
        if (lane == 0) qs[c] = on ? s : -1.0f;  // -1 marks a padding column
    }
    __syncthreads();

    const int rows_per_tile = sh.cols_per_row < 8 ? 8 / sh.cols_per_row : 1;  // rows in an 8-column tile
    float best[2] = {kNegInf, kNegInf};
    for (int c0 = 0; c0 < cols; c0 += 8) {
        int acc[4] = {0, 0, 0, 0};
        const uint4* bq = reinterpret_cast<const uint4*>(q8 + (c0 + g) * kStride) + t;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint4 w = bq[4 * i];
            const uint32_t a0[4] = {lo4[i].x, hi4[i].x, lo4[i].y, hi4[i].y};
            const uint32_t a1[4] = {lo4[i].z, hi4[i].z, lo4[i].w, hi4[i].w};
            mma_s8(acc, a0, w.x, w.y);
            mma_s8(acc, a1, w.z, w.w);
        }
        // acc: blocks g, g + 8 x columns 2t, 2t + 1
        float v[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float s = qs[c0 + 2 * t + e];
#pragma unroll
            for (int r = 0; r < 2; ++r)
                v[r][e] = s < 0.0f ? kNegInf : __fmul_rn(static_cast<float>(acc[2 * r + e]), s);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (sh.cols_per_row >= 2) v[r][0] = v[r][1] = fmaxf(v[r][0], v[r][1]);
            if (sh.cols_per_row >= 4) v[r][0] = v[r][1] = fmaxf(v[r][0], __shfl_xor_sync(kFull, v[r][0], 1));
            if (sh.cols_per_row >= 8) v[r][0] = v[r][1] = fmaxf(v[r][0], __shfl_xor_sync(kFull, v[r][0], 2));
        }
        bool last = true;
        if (sh.cols_per_row > 8) {  // a row of several tiles
            const int part = (c0 / 8) % (sh.cols_per_row / 8);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                best[r] = part == 0 ? v[r][0] : fmaxf(best[r], v[r][0]);
                v[r][0] = best[r];
            }
            last = part == sh.cols_per_row / 8 - 1;
        }
        if (!last) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = 2 * t + e;
            // one writer per row of the tile: its first column
            if (sh.cols_per_row >= 8 ? col != 0 : col % sh.cols_per_row != 0) continue;
            const int r = sh.cols_per_row >= 8 ? c0 / sh.cols_per_row : c0 / 8 * rows_per_tile + col / sh.cols_per_row;
            if (r0 + r >= r1) continue;
            float* out = scores + (static_cast<size_t>(first + r0 + r) * cache.n_kv_heads + head) * sh.stride;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int b = b0 + warp * 16 + g + 8 * k;
                if (b < row_blocks(len, n, r0 + r)) out[b] = page[k] < 0 ? kNegInf : __fmul_rn(v[k][e], scale[k]);
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

__global__ void __launch_bounds__(kPickThreads) kv_pick_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                               gofann_kv_select_params p, uint32_t stride,
                                                               const float* __restrict__ scores)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t warp_sum[kPickThreads / 32][2];
    __shared__ uint32_t found_digit, found_rank;
    const uint32_t row = blockIdx.x, head = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t seq = 0, at = 0;
    const auto rows = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>(n);
    };
    int blocks = 0;
    if (kv_find(batch.n_seqs, row, rows, seq, at)) {
        int first, n;
        kv_rows(batch, seq, first, n);
        blocks = row_blocks(kv_len(batch, seq), n, static_cast<int>(at));
    }
    const float* sc = scores + (static_cast<size_t>(row) * cache.n_kv_heads + head) * stride;
    int32_t* ids = p.ids + (static_cast<size_t>(row) * cache.n_kv_heads + head) * p.n_select;
    float* out = p.scores ? p.scores + (static_cast<size_t>(row) * cache.n_kv_heads + head) * p.n_select : nullptr;
    const int want = static_cast<int>(p.n_select);
    const auto key_of = [&](int b) {
        const float x = sc[b];
        if (x == kNegInf) return 0u;
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
            if (out) out[slot] = sc[b];
        }
        __syncthreads();
    }
    const uint32_t filled = taken + (tied < ties ? tied : ties);
    for (uint32_t i = filled + threadIdx.x; i < static_cast<uint32_t>(want); i += kPickThreads) {
        ids[i] = -1;
        if (out) out[i] = kNegInf;
    }
}

SelectShape select_shape(const gofann_kv_cache& c, const gofann_kv_batch& b, const gofann_kv_select_params& p)
{
    SelectShape s;
    s.group = static_cast<int>(p.n_heads / c.n_kv_heads);
    int cols = 1;
    while (cols < 8 && cols < s.group) cols *= 2;
    s.cols_per_row = s.group > 8 ? (s.group + 7) / 8 * 8 : cols;
    s.rows_per_block = s.cols_per_row >= kScoreCols ? 1 : kScoreCols / s.cols_per_row;
    s.block_tiles = (b.max_pages + kScoreBlocks - 1) / kScoreBlocks;
    s.stride = (b.max_pages + 3) / 4 * 4;
    return s;
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
    if (batch->max_pages == 0) return fail(GOFANN_ERR_INVALID, "kv_select: rows without pages");
    const size_t need = gofann_kv_select_scratch_bytes(cache, batch, params);
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255))
        return fail(GOFANN_ERR_INVALID, "kv_select: scratch must be 256-byte aligned");
    if (scratch_bytes < need)
        return fail(GOFANN_ERR_CAPACITY, "kv_select: scratch of %zu bytes, %zu needed", scratch_bytes, need);
    const SelectShape s = select_shape(*cache, *batch, p);
    // a sequence of n rows has at most n / rows_per_block + 1 tiles, and at most n
    const uint64_t bound = static_cast<uint64_t>(batch->n_rows) / s.rows_per_block + batch->n_seqs;
    const uint64_t tiles = (bound < batch->n_rows ? bound : batch->n_rows) * s.block_tiles;
    if (tiles > 0x7fffffffull)
        return fail(GOFANN_ERR_UNSUPPORTED, "kv_select: %llu tiles (at most 2^31 - 1)", static_cast<unsigned long long>(tiles));
    float* scores = static_cast<float*>(scratch);
    cudaStream_t cs = as_stream(stream);
    const dim3 grid(static_cast<uint32_t>(tiles), cache->n_kv_heads);
    const size_t cols = static_cast<size_t>(s.rows_per_block) * s.cols_per_row;
    const size_t smem = cols * (2 * d + 16 + 4);
    if (smem > 200 * 1024)
        return fail(GOFANN_ERR_UNSUPPORTED, "kv_select: %d query heads per key/value head", s.group);
    const void* fn = d == 64 ? reinterpret_cast<const void*>(kv_score_kernel<64>)
                             : reinterpret_cast<const void*>(kv_score_kernel<128>);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return cuda_status(e, "kv_select: shared memory attribute");
    }
    if (d == 64)
        kv_score_kernel<64><<<grid, kScoreThreads, smem, cs>>>(*cache, *batch, p, s, scores);
    else
        kv_score_kernel<128><<<grid, kScoreThreads, smem, cs>>>(*cache, *batch, p, s, scores);
    GOFANN_CHECK_LAUNCH("kv_score_kernel");
    kv_pick_kernel<<<dim3(batch->n_rows, cache->n_kv_heads), kPickThreads, 0, cs>>>(*cache, *batch, p, s.stride, scores);
    GOFANN_CHECK_LAUNCH("kv_pick_kernel");
    return GOFANN_OK;
}

}  // extern "C"
