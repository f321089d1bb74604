// kv_attention_rows.cu — attention over the 4-bit cache for many query rows:
// the products of 256 query columns with 128 tokens at a time on the 5th
// generation tensor cores.
//
// A block has two tiles of 128 query columns (token rows x query heads of one
// key/value head) and walks their blocks of the cache, two pages (128 tokens)
// a step:
// * a loader copies packed chunks to a shared ring (bulk copies);
// * four warps turn codes into f16 keys [token][dim] and transposed values
//   [dim][token], both 128-byte swizzled and K-major, each page once for all
//   256 columns;
// * one thread issues S = Q K^T (tcgen05.mma, M = 128, N = 128) and
//   O += P V (M = 128, N = head_dim, P from tensor memory);
// * two warpgroups, one thread a query column, turn S into P: maximum, mask,
//   exponential; P takes the place of S in tensor memory as f16.
// While one tile is in the exponentials the other has the tensor cores.
//
// Precision: keys and values c * s + m are rounded to f16 (at most 2^-11 of
// the value; a quantisation step is at least 2^-4 of the group's range, so
// this is below 2^-7 of what the cache has already rounded), weights to f16;
// logits, maxima, sums and the output are f32.  The reference point of a
// column's weights follows its maximum only once it is 2^8 behind, so the
// output is rarely rescaled; weights are at most 2^15, which f16 holds.
#include "kv_attention.cuh"

namespace gofann {
namespace {

constexpr int kTileRows = 128, kTiles = 2;
constexpr int kStepKeys = 2 * kKvPage;
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4;  // a decode warp has a quarter of every group
constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps, kLoadWarp = kMmaWarp + 1;
constexpr int kRowThreads = 32 * (kLoadWarp + 1);
constexpr float kLag = 8.0f;   // log2 that a column's maximum may run ahead of its reference
constexpr float kHead = 7.0f;  // log2 of a weight at the reference

template <int D>
struct Rows {
    static constexpr int kPanels = D / 64;                          // 64 dimensions = one 128-byte swizzled row
    static constexpr int kQTile = kTileRows * D * 2;
    static constexpr int kKeys = kStepKeys * D * 2;                 // [panel][128 tokens][64 dims]
    static constexpr int kValues = kStepKeys * D * 2;               // [page][D dims][64 tokens]
    static constexpr int kChunk = KvChunk<D>::kBytes;
    static constexpr int kRaw = D == 64 ? 6 : 3;
    static constexpr int kOffK = kTiles * kQTile;
    static constexpr int kOffV = kOffK + 2 * kKeys;
    static constexpr int kOffRaw = kOffV + 2 * kValues;
    static constexpr int kOffShown = kOffRaw + kRaw * kChunk;       // u64 [kRaw] of the ring, [4][2] of the steps
    static constexpr int kOffBars = kOffShown + 8 * (kRaw + 8);
    static constexpr int kBars = 2 * kRaw + 8 + 3 * kTiles + 2;
    static constexpr int kBytes = 1024 + kOffBars + 8 * kBars + 16;
    static_assert(kBytes <= 227 * 1024, "shared memory of a block");
    // tensor memory columns
    static constexpr uint32_t kScores = 0, kOut = kTiles * kStepKeys, kColumns = 512;
};

// ------------------------------------------------------------ tensor cores
// Shared-memory descriptor of a K-major operand in 128-byte swizzled rows
// (8-row atoms 1024 bytes apart).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr)
{
    uint64_t d = static_cast<uint64_t>((addr & 0x3ffffu) >> 4);
    d |= 1ull << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}
// Instruction descriptor: f32 += f16 x f16, both K-major.
__host__ __device__ constexpr uint32_t mma_shape(int m, int n)
{
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t add)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(add)
        : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, uint32_t add)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"(add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of this thread's lane; the values are there after
// tensor_wait_load and tensor_ready.
__device__ __forceinline__ void tensor_load(uint32_t addr, float* v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tensor_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Orders the uses of 32 loaded values behind the wait.
__device__ __forceinline__ void tensor_ready(float* v)
{
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                   "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                   "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                   "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ __forceinline__ void tensor_store(uint32_t addr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
        "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tensor_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 numbers in one 64-bit register, for instructions on both.
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float first_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float second_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// ------------------------------------------------------------------ decoding
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// The pairs of codes in the low and high nibbles of bytes 0 and 2, as f16
// numbers: 0x6400 | c is 1024 + c, 0x6400 | 16 c is 1024 + 16 c, both exact.
__device__ __forceinline__ void code_pairs(uint32_t w, __half2& low, __half2& high)
{
    const __half2 minus = as_half2(0xe400e400u), sixteenth = as_half2(0x2c002c00u), back = as_half2(0xd400d400u);
    low = __hadd2(as_half2((w & 0x000f000fu) | 0x64006400u), minus);              // - 1024
    high = __hfma2(as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, back);  // / 16 - 64
}

// Keys of one page: this warp's quarter (16 tokens) as rows of 64 dimensions.
template <int D>
__device__ __forceinline__ void decode_keys(const unsigned char* chunk, unsigned char* keys, int page, int warp)
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, kt = warp;
    const int token0 = 16 * (g >> 1) + 4 * kt + (g & 1);
    const uint32_t* params = reinterpret_cast<const uint32_t*>(chunk + KvChunk<D>::kKeyParams) + (g * 4 + kt) * 2 * G;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
        const uint4 w4 = reinterpret_cast<const uint4*>(chunk)[(kt * G + grp) * 32 + lane];
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const __half2 sm = as_half2(params[r * G + grp]);
            const __half2 s = __low2half2(sm), m = __high2half2(sm);
            uint32_t out[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                __half2 a, b;
                code_pairs(r ? w[j] >> 8 : w[j], a, b);
                out[2 * j] = as_word(__hfma2(a, s, m));
                out[2 * j + 1] = as_word(__hfma2(b, s, m));
            }
            const int row = page * kKvPage + token0 + 2 * r;
            unsigned char* dst = keys + grp * (kStepKeys * 128) + row * 128;
            *reinterpret_cast<uint4*>(dst + (((2 * t) ^ (row & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<uint4*>(dst + (((2 * t + 1) ^ (row & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
        }
    }
}

// Values of one page, transposed: this warp's 16-dimension tiles as rows of 64
// tokens.  A hidden token's value is 0 whatever the page holds there.
template <int D>
__device__ __forceinline__ void decode_values(const unsigned char* chunk, unsigned char* values, int warp, uint64_t shown)
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // scales and minima of this lane's 16 tokens 16 t .. 16 t + 15, in pairs
    __half2 s[G][8], m[G][8];
    {
        const uint4* params = reinterpret_cast<const uint4*>(chunk + KvChunk<D>::kValueParams) + t * 4 * G;
#pragma unroll
        for (int q = 0; q < 2 * G; ++q) {
            const uint4 a4 = params[q], b4 = params[2 * G + q];  // even, odd tokens
            uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = (4 * q + k) / G, grp = (4 * q + k) % G;  // tokens 16 t + 2 i, + 1
                if (shown != ~0ull) {
                    const uint32_t two = static_cast<uint32_t>(shown >> (16 * t + 2 * i));
                    if (!(two & 1u)) a[k] = 0;
                    if (!(two & 2u)) b[k] = 0;
                }
                s[grp][i] = as_half2(__byte_perm(a[k], b[k], 0x5410));
                m[grp][i] = as_half2(__byte_perm(a[k], b[k], 0x7632));
            }
        }
    }
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
        {
            const int i = 4 * grp + warp;
            const uint4 w4 = reinterpret_cast<const uint4*>(chunk + KvChunk<D>::kValueCodes)[i * 32 + lane];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                uint32_t out[8];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    __half2 a, b;
                    code_pairs(r ? w[kt] >> 8 : w[kt], a, b);
                    out[2 * kt] = as_word(__hfma2(a, s[grp][2 * kt], m[grp][2 * kt]));
                    out[2 * kt + 1] = as_word(__hfma2(b, s[grp][2 * kt + 1], m[grp][2 * kt + 1]));
                }
                const int row = 16 * i + 8 * r + g;
                unsigned char* dst = values + row * 128;
                *reinterpret_cast<uint4*>(dst + (((2 * t) ^ (row & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4*>(dst + (((2 * t + 1) ^ (row & 7)) << 4)) =
                    make_uint4(out[4], out[5], out[6], out[7]);
            }
        }
    }
}

// ------------------------------------------------------------------ the kernel
template <int D>
__global__ void __launch_bounds__(kRowThreads, 1) kv_attend_rows_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                        gofann_kv_attention_params p, bool wide)
{
    using Cfg = Rows<D>;
    constexpr int kRaw = Cfg::kRaw;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* raw_shown = reinterpret_cast<uint64_t*>(smem + Cfg::kOffShown);  // [kRaw]
    uint64_t* step_shown = raw_shown + kRaw;                                   // [4][2]
    const uint32_t bars = shared_addr(smem + Cfg::kOffBars);
    const uint32_t raw_full = bars, raw_empty = raw_full + 8 * kRaw;
    const uint32_t k_full = raw_empty + 8 * kRaw, k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 16;
    const uint32_t s_full = v_empty + 16, p_full = s_full + 8 * kTiles, o_done = p_full + 8 * kTiles;
    const uint32_t q_full = o_done + 8 * kTiles, all_done = q_full + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffBars + 8 * Cfg::kBars);
    volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);  // a wait has run out

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const uint32_t head = blockIdx.y;
    // the sequence's last columns see most under a causal mask: they go first
    uint32_t seq, tile_at;
    const auto tiles = [&](uint32_t s) {
        int first, n;
        kv_rows(batch, s, first, n);
        return static_cast<uint32_t>((n * group + kTiles * kTileRows - 1) / (kTiles * kTileRows));
    };
    if (!kv_find<uint32_t>(batch.n_seqs, gridDim.x - 1 - blockIdx.x, tiles, seq, tile_at)) return;
    int first_row, n_rows;
    kv_rows(batch, seq, first_row, n_rows);
    const int len = kv_len(batch, seq);
    const int col0 = static_cast<int>(tile_at) * kTiles * kTileRows, total = n_rows * group;
    const int cols = total - col0 < kTiles * kTileRows ? total - col0 : kTiles * kTileRows;
    int lo, hi;
    dense_blocks(p, group, len, n_rows, col0, cols, lo, hi);
    const int pages = hi - lo, steps = (pages + 1) / 2;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRaw; ++i) {
            barrier_init(raw_full + 8 * i, 1);
            barrier_init(raw_empty + 8 * i, kDecodeWarps);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(k_full + 8 * i, kDecodeWarps);
            barrier_init(k_empty + 8 * i, 1);
            barrier_init(v_full + 8 * i, kDecodeWarps);
            barrier_init(v_empty + 8 * i, 1);
        }
        for (int i = 0; i < kTiles; ++i) {
            barrier_init(s_full + 8 * i, 1);
            barrier_init(p_full + 8 * i, kTileRows);
            barrier_init(o_done + 8 * i, 1);
        }
        barrier_init(q_full, kTiles * kTileRows);
        barrier_init(all_done, 1);
        barrier_fence();
        *dead = 0;
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)),
                     "r"(Cfg::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    const auto wait = [&](uint32_t bar, uint32_t parity) {
        if (*dead) return false;
        if (barrier_wait(bar, parity & 1)) return true;
        *dead = 1;
        return false;
    };

    if (warp == kLoadWarp) {
        // ---- loader: page numbers are looked up 32 blocks at a time
        int page = -1, issued = 0;
        uint64_t shown = 0;
        for (int i = 0; i < 2 * steps; ++i) {
            if ((i & 31) == 0) {
                const int block = lo + i + lane;
                page = -1;
                shown = 0;
                if (block < hi) {
                    page = __ldg(batch.page_table + static_cast<size_t>(seq) * batch.max_pages + block);
                    if (page < 0 || static_cast<uint32_t>(page) >= cache.n_pages) {
                        page = -1;
                        kv_invalid(batch);
                    } else {
                        shown = shown_tokens(p, seq, len, block);
                    }
                }
            }
            const int slot = i % kRaw;
            const int from = __shfl_sync(kFull, page, i & 31);
            const uint64_t bits = __shfl_sync(kFull, shown, i & 31);
            if (i >= kRaw && !wait(raw_empty + 8 * slot, i / kRaw - 1)) break;
            if (lane == 0) {
                raw_shown[slot] = bits;
                if (from >= 0) {
                    barrier_expect(raw_full + 8 * slot, Cfg::kChunk);
                    bulk_load(shared_addr(smem + Cfg::kOffRaw + slot * Cfg::kChunk),
                              cache.pages + (static_cast<size_t>(from) * cache.n_kv_heads + head) * Cfg::kChunk, Cfg::kChunk,
                              raw_full + 8 * slot);
                } else {
                    barrier_arrive(raw_full + 8 * slot);
                }
            }
            issued = i + 1;
        }
        // copies in flight may not outlive the block's shared memory
        for (int i = issued > kRaw ? issued - kRaw : 0; i < issued; ++i)
            if (!barrier_wait(raw_full + 8 * (i % kRaw), (i / kRaw) & 1)) *dead = 1;
    } else if (warp == kMmaWarp) {
        // ---- products, issued by one thread; the tensor cores take them in
        // order, so a tile's next S may be issued behind the product that
        // still reads its P
        if (lane == 0 && steps > 0) {
            const uint32_t base = shared_addr(smem);
            const auto scores = [&](int tile, int j) {
                const uint32_t q = base + tile * Cfg::kQTile, k = base + Cfg::kOffK + (j & 1) * Cfg::kKeys;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    mma_shared(tmem + Cfg::kScores + tile * kStepKeys,
                               operand_desc(q + (i / 4) * (kTileRows * 128) + (i % 4) * 32),
                               operand_desc(k + (i / 4) * (kStepKeys * 128) + (i % 4) * 32), mma_shape(kTileRows, kStepKeys),
                               i > 0);
                mma_commit(s_full + 8 * tile);
            };
            bool ok = wait(q_full, 0) && wait(k_full, 0);
            if (ok) {
                fence_after();
                for (int tile = 0; tile < kTiles; ++tile) scores(tile, 0);
                mma_commit(k_empty);
            }
            for (int j = 0; j < steps && ok; ++j) {
                for (int tile = 0; tile < kTiles && ok; ++tile) {
                    if (tile == 0) ok = wait(v_full + 8 * (j & 1), j >> 1);
                    ok = ok && wait(p_full + 8 * tile, j);
                    if (!ok) break;
                    fence_after();
                    const uint32_t v = base + Cfg::kOffV + (j & 1) * Cfg::kValues;
#pragma unroll
                    for (int i = 0; i < kStepKeys / 16; ++i)
                        mma_tensor(tmem + Cfg::kOut + tile * D, tmem + Cfg::kScores + tile * kStepKeys + 8 * i,
                                   operand_desc(v + (i / 4) * (D * 128) + (i % 4) * 32), mma_shape(kTileRows, D),
                                   j > 0 || i > 0);
                    mma_commit(o_done + 8 * tile);
                    if (tile == kTiles - 1) mma_commit(v_empty + 8 * (j & 1));
                    if (j + 1 < steps) {
                        if (tile == 0) {
                            ok = wait(k_full + 8 * ((j + 1) & 1), (j + 1) >> 1);
                            if (!ok) break;
                            fence_after();
                        }
                        scores(tile, j + 1);
                        if (tile == kTiles - 1) mma_commit(k_empty + 8 * ((j + 1) & 1));
                    }
                }
            }
            mma_commit(all_done);
            if (!barrier_wait(all_done, 0)) *dead = 1;
        }
        __syncwarp();
    } else if (warp >= kSoftmaxWarps) {
        // ---- codes to f16 operands
        const int w = warp - kSoftmaxWarps;
        for (int j = 0; j < steps; ++j) {
            const int st = j & 1;
            if (j >= 2 && !wait(k_empty + 8 * st, (j >> 1) - 1)) break;
            unsigned char* keys = smem + Cfg::kOffK + st * Cfg::kKeys;
            unsigned char* values = smem + Cfg::kOffV + st * Cfg::kValues;
            bool ok = true;
            for (int h = 0; h < 2 && ok; ++h) {
                const int i = 2 * j + h, slot = i % kRaw;
                ok = wait(raw_full + 8 * slot, i / kRaw);
                if (!ok) break;
                decode_keys<D>(smem + Cfg::kOffRaw + slot * Cfg::kChunk, keys, h, w);
                if (w == 0 && lane == 0) step_shown[(j & 3) * 2 + h] = raw_shown[slot];
            }
            if (!ok) break;
            fence_shared();
            __syncwarp();
            if (lane == 0) barrier_arrive(k_full + 8 * st);
            if (j >= 2 && !wait(v_empty + 8 * st, (j >> 1) - 1)) break;
            for (int h = 0; h < 2; ++h) {
                const int slot = (2 * j + h) % kRaw;
                decode_values<D>(smem + Cfg::kOffRaw + slot * Cfg::kChunk, values + h * (D * 128), w, raw_shown[slot]);
                __syncwarp();
                if (lane == 0) barrier_arrive(raw_empty + 8 * slot);
            }
            fence_shared();
            __syncwarp();
            if (lane == 0) barrier_arrive(v_full + 8 * st);
        }
    } else {
        // ---- softmax: one thread a query column
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const int col = tile * kTileRows + row;
        const bool on = col < cols;
        const int at_col = col0 + (on ? col : 0);
        const uint64_t out_row =
            static_cast<uint64_t>(first_row + at_col / group) * p.n_heads + head * group + at_col % group;
        int low, limit;
        row_limits(p, len - n_rows + at_col / group, len, low, limit);
        float unit = 1.0f;
        {
            const uint64_t src = static_cast<uint64_t>(first_row + at_col / group) * p.q_stride +
                                 static_cast<uint64_t>(head * group + at_col % group) * D;
            float top = 0.0f;
#pragma unroll 8
            for (int d = 0; d < D; d += 4) {
                float x[4];
                kv_load4(p.q, src + d, p.dtype, wide, x);
                top = fmaxf(fmaxf(fmaxf(top, fabsf(x[0])), fmaxf(fabsf(x[1]), fabsf(x[2]))), fabsf(x[3]));
            }
            const int ex = query_exponent(top);
            // a negative scale turns the query around, a scale of 0 makes it 0
            const float down = on ? power_of_two(ex) * (p.scale < 0.0f ? -1.0f : p.scale > 0.0f ? 1.0f : 0.0f) : 0.0f;
            if (p.scale != 0.0f) unit = fmaxf(fabsf(p.scale) * kLog2e * power_of_two(-ex), FLT_MIN);
            unsigned char* q = smem + tile * Cfg::kQTile + row * 128;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                float x[4], y[4];
                kv_load4(p.q, src + d, p.dtype, wide, x);
                kv_load4(p.q, src + d + 4, p.dtype, wide, y);
                const uint4 w = make_uint4(as_word(__floats2half2_rn(x[0] * down, x[1] * down)),
                                           as_word(__floats2half2_rn(x[2] * down, x[3] * down)),
                                           as_word(__floats2half2_rn(y[0] * down, y[1] * down)),
                                           as_word(__floats2half2_rn(y[2] * down, y[3] * down)));
                *reinterpret_cast<uint4*>(q + (d / 64) * (kTileRows * 128) + (((d % 64 / 8) ^ (row & 7)) << 4)) = w;
            }
            fence_shared();
            barrier_arrive(q_full);
        }
        // keys in (warp_low, warp_limit] are seen by every column of the warp
        const int warp_limit = __reduce_min_sync(kFull, on ? limit : 0x7fffffff);
        const int warp_low = __reduce_max_sync(kFull, on ? low : -1);

        const uint32_t s_at = tmem + lanes + Cfg::kScores + tile * kStepKeys, o_at = tmem + lanes + Cfg::kOut + tile * D;
        float ref = kNegInf;
        uint64_t l2 = 0;  // two parts of the sum of weights
        bool ok = true;
        for (int j = 0; j < steps; ++j) {
            ok = wait(s_full + 8 * tile, j);
            if (!ok) break;
            fence_after();
            const int key0 = (lo + 2 * j) * kKvPage;
            const uint64_t shown[2] = {step_shown[(j & 3) * 2], step_shown[(j & 3) * 2 + 1]};
            const bool masked = (shown[0] & shown[1]) != ~0ull || key0 + kStepKeys - 1 > warp_limit || key0 <= warp_low;
            if (masked) {
                // hidden tokens' scores become -inf in place; the rest of the
                // step then knows no mask
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int a = limit - (key0 + 32 * c), b = low - (key0 + 32 * c);
                    uint32_t see = static_cast<uint32_t>(shown[c >> 1] >> (32 * (c & 1)));
                    see &= a < 0 ? 0u : a >= 31 ? ~0u : (2u << a) - 1u;
                    see &= b < 0 ? ~0u : b >= 31 ? 0u : ~((2u << b) - 1u);
                    float v[32];
                    tensor_load(s_at + 32 * c, v);
                    tensor_wait_load();
                    tensor_ready(v);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!((see >> i) & 1)) v[i] = kNegInf;
                    tensor_store(s_at + 32 * c, reinterpret_cast<const uint32_t*>(v));
                }
                tensor_wait_store();
            }
            float v[64];
            float mx = kNegInf;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                tensor_load(s_at + 64 * c, v);
                tensor_load(s_at + 64 * c + 32, v + 32);
                tensor_wait_load();
                tensor_ready(v);
                tensor_ready(v + 32);
                float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < 64; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) m4[k] = i + 4 + k < 64 ? fmaxf(fmaxf(m4[k], v[i + k]), v[i + 4 + k]) : fmaxf(m4[k], v[i + k]);
                mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
            }
            // the reference follows the maximum where that is far ahead
            float f = 1.0f;
            if (ref == kNegInf) {
                ref = mx;
            } else if ((mx - ref) * unit > kLag) {
                f = exp2_fast((ref - mx) * unit);
                ref = mx;
                l2 = fma_two(l2, pair(f, f), 0);
            }
            if (__any_sync(kFull, f != 1.0f)) {
                ok = wait(o_done + 8 * tile, j - 1);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    tensor_load(o_at + 32 * c, o);
                    tensor_wait_load();
                    tensor_ready(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f;
                    tensor_store(o_at + 32 * c, reinterpret_cast<const uint32_t*>(o));
                }
            }
            const float minus_base = fmaf(ref == kNegInf ? 0.0f : -ref, unit, kHead);
            const uint64_t unit2 = pair(unit, unit), minus_base2 = pair(minus_base, minus_base);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                tensor_load(s_at + 64 * c, v);
                tensor_load(s_at + 64 * c + 32, v + 32);
                tensor_wait_load();
                tensor_ready(v);
                tensor_ready(v + 32);
                uint32_t w[32];
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const uint64_t x = fma_two(pair(v[i], v[i + 1]), unit2, minus_base2);
                    const float a = exp2_fast(first_of(x)), b = exp2_fast(second_of(x));
                    sum[(i >> 1) & 1] = add_two(sum[(i >> 1) & 1], pair(a, b));
                    w[i / 2] = as_word(__floats2half2_rn(a, b));
                }
                l2 = add_two(l2, add_two(sum[0], sum[1]));
                // P takes the columns of S that have been read
                tensor_store(s_at + 32 * c, w);
            }
            tensor_wait_store();
            fence_before();
            barrier_arrive(p_full + 8 * tile);
        }
        // ---- the output of this thread's column
        if (ok && steps > 0) {
            ok = wait(o_done + 8 * tile, steps - 1);
            fence_after();
        }
        if (ok) {
            const float l = first_of(l2) + second_of(l2), inv = l > 0.0f ? 1.0f / l : 0.0f;
            uint16_t* out = static_cast<uint16_t*>(p.out) + out_row * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                if (steps > 0) {
                    tensor_load(o_at + 32 * c, o);
                    tensor_wait_load();
                    tensor_ready(o);
                }
                if (on) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        uint2 w = make_uint2(0u, 0u);
                        if (l > 0.0f)
                            w = make_uint2(kv_pack2(o[i] * inv, o[i + 1] * inv, p.dtype),
                                           kv_pack2(o[i + 2] * inv, o[i + 3] * inv, p.dtype));
                        *reinterpret_cast<uint2*>(out + 32 * c + i) = w;
                    }
                }
            }
            if (on && p.lse)
                p.lse[out_row] = l > 0.0f ? (fmaf(ref, unit, -kHead) + log2f(l)) * kLn2 : kNegInf;
            fence_before();
        }
    }

    // every product has completed (or its wait has run out) before the tensor
    // memory goes back
    __syncthreads();
    if (threadIdx.x == 0 && *dead) kv_timeout(batch);
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kColumns) : "memory");
    }
}

template <int D>
int launch_rows(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                cudaStream_t s)
{
    const uint64_t group = p.n_heads / cache.n_kv_heads, width = kTiles * kTileRows;
    // a sequence of n rows has at most n group / width + 1 tiles, and at most one per column
    const uint64_t cols = static_cast<uint64_t>(batch.n_rows) * group;
    uint64_t tiles = cols / width + batch.n_seqs;
    if (tiles > cols) tiles = cols;
    if (tiles > 0x7fffffffull)
        return fail(GOFANN_ERR_UNSUPPORTED, "kv_attention: %llu tiles (at most 2^31 - 1)", static_cast<unsigned long long>(tiles));
    auto* kernel = kv_attend_rows_kernel<D>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Rows<D>::kBytes);
    if (e != cudaSuccess) return cuda_status(e, "kv_attention: shared memory attribute");
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && (p.q_stride & 3) == 0;
    kernel<<<dim3(static_cast<uint32_t>(tiles), cache.n_kv_heads), kRowThreads, Rows<D>::kBytes, s>>>(cache, batch, p, wide);
    GOFANN_CHECK_LAUNCH("kv_attend_rows_kernel");
    return GOFANN_OK;
}

}  // namespace

int attend_rows(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                cudaStream_t s)
{
    return cache.head_dim == 64 ? launch_rows<64>(cache, batch, p, s) : launch_rows<128>(cache, batch, p, s);
}

}  // namespace gofann
