// kv_attention_rows.cu — attention over the 4-bit cache for many query rows:
// the products of 256 query columns with 128 tokens at a time on the 5th
// generation tensor cores.
//
// A block takes two tiles of 128 query columns (token rows x query heads of
// one key/value head) at a time and walks their blocks of the cache, two pages
// (128 tokens) a step:
// * a loader copies packed chunks to a shared ring (bulk copies);
// * eight warps turn codes into keys [token][dim], each a sum of two f16
//   numbers, and four into f16 values [dim][token], all 128-byte swizzled and
//   K-major, each page once for all 256 columns;
// * one thread issues S = Q K^T (tcgen05.mma, M = 128, N = 128, twice: the
//   keys' upper and lower parts) and O += P V (M = 128, N = head_dim, P from
//   tensor memory);
// * two warpgroups, one thread a query column, turn S into P: mask and
//   exponential; P takes the place of S in tensor memory as f16.
// While one tile is in the exponentials the other has the tensor cores.
//
// What bounds it: the tensor cores' products (the keys' lower
// parts are a third of them), whose operands share shared memory's port with the
// decoded pages and tensor memory's with S and P.  Chunks of 2043 rows of two
// prompts (32 query, 8 key/value heads of 128, up to 12289 tokens): 686
// GFLOP of visible products in 1315 us, 522 TFLOP/s, 0.31 of a plain product's
// measured rate; the tensor pipe is active 40 % of the time, and the thread
// that issues waits 0.4 of a step: for P 1850 of 7500 cycles, for values 510,
// for keys 430.  Keys of one f16 number took 900 us.  Eight warps for values,
// values decoded before their buffer is free, one lane a warp that waits or
// arrives: no gain.
//
// The steps of all items (256 columns, head) are dealt out evenly, one block
// per SM: a block does a run of them, and an item that a share's end cuts is
// joined from partial results by a second, programmatic launch.
//
// Precision: a key c * s + m is held as its f16 rounding and the f16 rounding
// of what that left, 22 bits in all: a logit that one f16 number a key gives
// is off by some 2e-4, which lse shows (up to 5e-5 of it where a row sees few
// tokens).  Values and weights are rounded to f16 once (2^-11; the output is
// of 16 bits anyway); logits, sums and the output are f32.  A column's weights are relative to a
// reference, its first maximum, times 2^7; the reference moves up to the
// maximum only where 32 weights sum to more than 2^15 (f16 ends at 2^16), so
// the maximum is rarely looked for and the output rarely rescaled.  The output
// leaves tensor memory for an f32 sum every 8192 tokens (kFold), as the tensor
// cores' own sum of values of one sign drifts (chunks of two prompts 1306 ->
// 1315 us).
#include "kv_attention.cuh"

namespace gofann {
namespace {

constexpr int kTileRows = 128, kTiles = 2;
constexpr int kStepKeys = 2 * kKvPage;
// Eight warps decode keys, a quarter of one of a step's two pages each; four
// decode values, a quarter of both.
constexpr int kSoftmaxWarps = 8, kKeyWarps = 8, kDecodeWarps = kKeyWarps + 4;
constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps, kLoadWarp = kMmaWarp + 1;
constexpr int kRowThreads = 32 * (kLoadWarp + 3);  // whole warpgroups
// Registers a thread: 80 at launch for 768 threads, 61440 in all, which is
// what 256 x 104 + 384 x 72 + 128 x 56 takes.
constexpr int kSoftmaxRegs = 104, kDecodeRegs = 72, kOtherRegs = 56;
constexpr float kHead = 7.0f;      // log2 of a weight at the reference
constexpr float kMost = 32768.0f;  // sum of 32 weights from which the reference moves up
// Steps after which the output so far leaves tensor memory.  The tensor cores
// truncate their sums, so a long one falls short: by 5e-8 of itself for every
// product of 16 tokens, 4e-4 over 131072 tokens (an f16's half unit is 2.4e-4
// to 4.9e-4).  512 products of 8192 tokens lose 2^-15 at the most; the parts
// are added in f32, rounded to nearest.
constexpr int kFold = 64;
static_assert((kFold & (kFold - 1)) == 0, "steps are counted modulo it");

template <int D>
struct Rows {
    static constexpr int kQTile = kTileRows * D * 2;
    static constexpr int kKeys = kStepKeys * D * 2;                 // [panel][128 tokens][64 dims]
    static constexpr int kValues = kStepKeys * D * 2;               // [page][D dims][64 tokens]
    static constexpr int kHalf = KvChunk<D>::kBytes / 2;            // keys or values of a page
    static constexpr int kRaw = D == 64 ? 12 : 6;
    // Stages of the keys' lower parts and of the values: what shared memory holds.
    static constexpr int kLate = D == 64 ? 2 : 1;
    static constexpr int kOffK = kTiles * kQTile;
    static constexpr int kOffLow = kOffK + 2 * kKeys;
    static constexpr int kOffV = kOffLow + kLate * kKeys;
    static constexpr int kOffRaw = kOffV + kLate * kValues;
    static constexpr int kOffShown = kOffRaw + kRaw * kHalf;        // u64 [8 steps][2 pages]
    static constexpr int kOffBars = kOffShown + 8 * 16;
    static constexpr int kBars = 2 * kRaw + 4 + 6 * kLate + 5 * kTiles + 2;
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
// d (+)= a b + a c: the second product takes a from the buffer that the first
// one left it in.
__device__ __forceinline__ void mma_shared_two(uint32_t d, uint64_t a, uint64_t b, uint64_t c, uint32_t shape, uint32_t add)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], %1, %2, %4, p;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], %1, %3, %4, q;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "l"(c), "r"(shape), "r"(add)
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
__device__ __forceinline__ void tensor_load16(uint32_t addr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tensor_store16(uint32_t addr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
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

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one()
{
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
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

// Two f32 numbers as f16, and what the rounding left of them.
__device__ __forceinline__ void split_two(uint64_t x, uint32_t& high, uint32_t& low)
{
    const __half2 h = __floats2half2_rn(first_of(x), second_of(x));
    const float2 back = __half22float2(h);
    const uint64_t rest = add_two(x, pair(-back.x, -back.y));
    high = as_word(h);
    low = as_word(__floats2half2_rn(first_of(rest), second_of(rest)));
}

// 16 bytes of every row of one page's keys: this warp's quarter (16 tokens) as
// rows of 64 dimensions.
template <int D>
__device__ __forceinline__ void store_keys(const uint32_t (&k)[KvChunk<D>::kGroups][2][8], unsigned char* keys, int page,
                                           int kt)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int token0 = 16 * (g >> 1) + 4 * kt + (g & 1);
#pragma unroll
    for (int grp = 0; grp < KvChunk<D>::kGroups; ++grp)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t(&w)[8] = k[grp][r];
            const int row = page * kKvPage + token0 + 2 * r;
            unsigned char* dst = keys + grp * (kStepKeys * 128) + row * 128;
            *reinterpret_cast<uint4*>(dst + (((2 * t) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(dst + (((2 * t + 1) ^ (row & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
}

// Keys of one page from the key half of its chunk, this warp's quarter, as
// sums of two f16 numbers: c * s + m takes up to 22 bits.
template <int D>
__device__ __forceinline__ void decode_keys(const unsigned char* chunk, int kt, uint32_t (&high)[KvChunk<D>::kGroups][2][8],
                                            uint32_t (&low)[KvChunk<D>::kGroups][2][8])
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const uint32_t* params = reinterpret_cast<const uint32_t*>(chunk + KvChunk<D>::kCodes) + (g * 4 + kt) * 2 * G;
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
        const uint4 w4 = reinterpret_cast<const uint4*>(chunk)[(kt * G + grp) * 32 + lane];
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float2 sm = __half22float2(as_half2(params[r * G + grp]));
            const uint64_t s2 = pair(sm.x, sm.x), m2 = pair(sm.y, sm.y);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                __half2 a, b;
                code_pairs(r ? w[j] >> 8 : w[j], a, b);
                const float2 x = __half22float2(a), y = __half22float2(b);
                split_two(fma_two(pair(x.x, x.y), s2, m2), high[grp][r][2 * j], low[grp][r][2 * j]);
                split_two(fma_two(pair(y.x, y.y), s2, m2), high[grp][r][2 * j + 1], low[grp][r][2 * j + 1]);
            }
        }
    }
}

// Values of one page from the value half, transposed: this warp's 16-dimension tiles as rows of 64
// tokens.  A hidden token's value is 0 whatever the page holds there.
template <int D>
__device__ __forceinline__ void decode_values(const unsigned char* chunk, unsigned char* values, int warp, uint64_t shown)
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // scales and minima of this lane's 16 tokens 16 t .. 16 t + 15, in pairs
    __half2 s[G][8], m[G][8];
    {
        const uint4* params = reinterpret_cast<const uint4*>(chunk + KvChunk<D>::kCodes) + t * 4 * G;
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
            const uint4 w4 = reinterpret_cast<const uint4*>(chunk)[i * 32 + lane];
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

// Weights 2^(unit x - base) of 32 scores as f16 pairs; returns their sum (two
// parts).
__device__ __forceinline__ uint64_t weigh(const float (&x)[32], float ref, float unit, uint32_t (&w)[16])
{
    const float minus_base = fmaf(ref == kNegInf ? 0.0f : -ref, unit, kHead);
    const uint64_t unit2 = pair(unit, unit), minus_base2 = pair(minus_base, minus_base);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const uint64_t y = fma_two(pair(x[i], x[i + 1]), unit2, minus_base2);
        const float a = exp2_fast(first_of(y)), b = exp2_fast(second_of(y));
        sum[(i >> 1) & 1] = add_two(sum[(i >> 1) & 1], pair(a, b));
        w[i / 2] = as_word(__floats2half2_rn(a, b));
    }
    return add_two(sum[0], sum[1]);
}
__device__ __forceinline__ float largest(const float (&x)[32])
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) m = fmaxf(m, x[i]);
    return m;
}

// 16 columns times f: f32 numbers of the output, or pairs of f16 weights.
// Rare, so kept out of the step's code.
__device__ __noinline__ void scale_output(uint32_t addr, float f)
{
    uint32_t r[16];
    tensor_load16(addr, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
    tensor_store16(addr, r);
}
__device__ __noinline__ void scale_weights(uint32_t addr, float f)
{
    uint32_t r[16];
    tensor_load16(addr, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 x = __half22float2(as_half2(r[i]));
        r[i] = as_word(__floats2half2_rn(x.x * f, x.y * f));
    }
    tensor_store16(addr, r);
}

// --------------------------------------------------------------- the schedule
constexpr int kWidth = kTiles * kTileRows;

// Work is counted in steps of one item (256 columns, key/value head); every
// item has at least one, so that it has an owner.
__device__ __forceinline__ int item_steps(const gofann_kv_attention_params& p, int group, int len, int n_rows, int tile)
{
    const int total = n_rows * group, col0 = tile * kWidth;
    int lo, hi;
    dense_blocks(p, group, len, n_rows, col0, total - col0 < kWidth ? total - col0 : kWidth, lo, hi);
    const int steps = (hi - lo + 1) / 2;
    return steps > 0 ? steps : 1;
}

// Where unit `flat` is (the warp's lanes share the tiles of a sequence), or
// with `flat` past the end the number of all units.
struct Place {
    uint32_t seq, head;
    int tile, step;
    uint64_t total;
};
__device__ __forceinline__ Place locate(const gofann_kv_batch& b, const gofann_kv_attention_params& p, uint32_t n_kv,
                                        int group, uint64_t flat)
{
    const int lane = threadIdx.x & 31;
    Place at{0, 0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < b.n_seqs; s0 += 32) {
        int first, n = 0, len = 0;
        if (s0 + lane < b.n_seqs) {
            kv_rows(b, s0 + lane, first, n);
            len = kv_len(b, s0 + lane);
        }
        for (int k = 0; k < 32 && s0 + k < b.n_seqs; ++k) {
            const int rows = __shfl_sync(kFull, n, k), length = __shfl_sync(kFull, len, k);
            const int tiles = (rows * group + kWidth - 1) / kWidth;
            uint64_t sum = 0;
            for (int i = lane; i < tiles; i += 32) sum += item_steps(p, group, length, rows, i);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
            if (sum == 0) continue;
            if (flat < sum * n_kv) {
                at.seq = s0 + k;
                at.head = static_cast<uint32_t>(flat / sum);
                uint64_t rest = flat % sum;
                for (int i0 = 0;; i0 += 32) {
                    const uint64_t c = i0 + lane < tiles ? item_steps(p, group, length, rows, i0 + lane) : 0;
                    uint64_t upto = c;
#pragma unroll
                    for (int off = 1; off < 32; off <<= 1) {
                        const uint64_t v = __shfl_up_sync(kFull, upto, off);
                        if (lane >= off) upto += v;
                    }
                    const unsigned past = __ballot_sync(kFull, rest < upto);
                    if (past) {
                        const int l = __ffs(past) - 1;
                        at.tile = i0 + l;
                        at.step = static_cast<int>(rest - __shfl_sync(kFull, upto - c, l));
                        return at;
                    }
                    rest -= __shfl_sync(kFull, upto, 31);
                }
            }
            flat -= sum * n_kv;
            at.total += sum * n_kv;
        }
    }
    return at;
}

// An item and the steps [from, to) of it that a block does.
struct Item {
    uint32_t seq, head;
    int tile, tiles;
    int first_row, n_rows, len, col0, cols;
    int lo, hi, steps, from, to;
    uint64_t flat, limit;  // units: where this part starts, where the block's share ends
};

__device__ __forceinline__ void open_item(const gofann_kv_batch& b, const gofann_kv_attention_params& p, int group, int step,
                                          Item& it)
{
    kv_rows(b, it.seq, it.first_row, it.n_rows);
    it.len = kv_len(b, it.seq);
    const int total = it.n_rows * group;
    it.tiles = (total + kWidth - 1) / kWidth;
    it.col0 = it.tile * kWidth;
    it.cols = total - it.col0 < kWidth ? total - it.col0 : kWidth;
    dense_blocks(p, group, it.len, it.n_rows, it.col0, it.cols, it.lo, it.hi);
    it.steps = item_steps(p, group, it.len, it.n_rows, it.tile);
    it.from = step;
    const uint64_t left = it.limit - it.flat;
    it.to = left < static_cast<uint64_t>(it.steps - step) ? step + static_cast<int>(left) : it.steps;
}
// The block's next item; false at the end of its share.
__device__ __forceinline__ bool next_item(const gofann_kv_batch& b, const gofann_kv_attention_params& p, uint32_t n_kv,
                                          int group, Item& it)
{
    it.flat += it.to - it.from;
    if (it.flat >= it.limit) return false;
    if (++it.tile == it.tiles) {
        it.tile = 0;
        if (++it.head == n_kv) {
            it.head = 0;
            int first, n = 0;
            while (n == 0 && it.seq + 1 < b.n_seqs) kv_rows(b, ++it.seq, first, n);
            if (n == 0) return false;
        }
    }
    open_item(b, p, group, 0, it);
    return true;
}

// Steps of one block: a share of the total, at least four (a partial result
// costs about as much as one step).
__device__ __forceinline__ uint64_t steps_per_block(uint64_t total, uint32_t blocks)
{
    const uint64_t c = (total + blocks - 1) / blocks;
    return c > 4 ? c : 4;
}

// A block's partial result in scratch: [256] base, [256] sum, [D][256]
// values, so that the threads of a warp, a column each, write side by side;
// two per block (its first item, and its last if that is another).  One more
// per block, behind those, is where its output is folded to: the reference of
// the weights in place of the base.
template <int D>
constexpr size_t kRowPartFloats = kWidth * (D + 2);

// Where this thread's column of a block's output is folded to.
template <int D>
__device__ __forceinline__ float* fold_column(float* parts)
{
    return parts + (2ull * gridDim.x + blockIdx.x) * kRowPartFloats<D> + threadIdx.x;
}
// The output so far, by the reference `ref`, joins what was folded before
// (unless it is the first); the next product starts it anew.  These are rare
// and kept out of the step's code, whose registers they would take.
template <int D>
__device__ __noinline__ void fold_output(uint32_t addr, float* parts, float ref, float unit, bool first)
{
    float* acc = fold_column<D>(parts);
    const float then = first ? kNegInf : *acc, f = then == kNegInf ? 0.0f : exp2_fast((then - ref) * unit);
    *acc = ref;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        uint32_t r[16];
        tensor_load16(addr + c, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float* at = acc + (2 + c + i) * kWidth;
            *at = f > 0.0f ? fmaf(*at, f, __uint_as_float(r[i])) : __uint_as_float(r[i]);
        }
    }
}
// What was folded joins the rest of the output in tensor memory.
template <int D>
__device__ __noinline__ void unfold_output(uint32_t addr, float* parts, float ref, float unit)
{
    const float* acc = fold_column<D>(parts);
    const float f = *acc == kNegInf ? 0.0f : exp2_fast((*acc - ref) * unit);
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        uint32_t r[16];
        tensor_load16(addr + c, r);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            r[i] = __float_as_uint(f > 0.0f ? fmaf(acc[(2 + c + i) * kWidth], f, __uint_as_float(r[i])) : __uint_as_float(r[i]));
        tensor_store16(addr + c, r);
    }
    tensor_wait_store();
}

// Place of a column's row in out and lse.
__device__ __forceinline__ uint64_t output_row(const gofann_kv_attention_params& p, int group, int first_row, uint32_t head,
                                               int col)
{
    return static_cast<uint64_t>(first_row + col / group) * p.n_heads + head * group + col % group;
}

// ------------------------------------------------------------------ the kernel
template <int D>
__global__ void __launch_bounds__(kRowThreads, 1) kv_attend_rows_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                        gofann_kv_attention_params p, bool wide,
                                                                        float* __restrict__ parts)
{
    using Cfg = Rows<D>;
    constexpr int kRaw = Cfg::kRaw;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Item start, warp_items[kSoftmaxWarps];  // of the softmax warps, to spare registers
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* step_shown = reinterpret_cast<uint64_t*>(smem + Cfg::kOffShown);  // [step & 7][page]
    const uint32_t bars = shared_addr(smem + Cfg::kOffBars);
    const uint32_t raw_full = bars, raw_empty = raw_full + 8 * kRaw;
    constexpr uint32_t kLate = Cfg::kLate;
    const uint32_t k_full = raw_empty + 8 * kRaw, k_empty = k_full + 16;
    const uint32_t low_full = k_empty + 16, low_empty = low_full + 8 * kLate;
    const uint32_t v_full = low_empty + 8 * kLate, v_empty = v_full + 16 * kLate;  // [stage][page]
    // [tile][half] of S and P
    const uint32_t s_full = v_empty + 16 * kLate, p_full = s_full + 16 * kTiles, q_full = p_full + 16 * kTiles;
    const uint32_t all_done = q_full + 8, o_half = all_done + 8;  // o_half: [tile] the first page's product
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffBars + 8 * Cfg::kBars);
    volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);  // a wait has run out

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const uint32_t n_kv = cache.n_kv_heads;
    launch_next();
    if (warp == 0) {
        const uint64_t total = locate(batch, p, n_kv, group, ~0ull).total;
        const uint64_t share = steps_per_block(total, gridDim.x), u0 = share * blockIdx.x;
        Item it{};
        if (u0 < total) {
            const Place at = locate(batch, p, n_kv, group, u0);
            it.seq = at.seq;
            it.head = at.head;
            it.tile = at.tile;
            it.flat = u0;
            it.limit = u0 + share < total ? u0 + share : total;
            open_item(batch, p, group, at.step, it);
        }
        if (lane == 0) start = it;
    }
    if (warp == 2 && blockIdx.x == 0) kv_check_sequences(batch, lane, 32);
    if (warp == 1 && lane == 0) {
        for (int i = 0; i < kRaw; ++i) {
            barrier_init(raw_full + 8 * i, 1);
            barrier_init(raw_empty + 8 * i, 4);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(k_full + 8 * i, kKeyWarps);
            barrier_init(k_empty + 8 * i, 1);
        }
        for (uint32_t i = 0; i < kLate; ++i) {
            barrier_init(low_full + 8 * i, kKeyWarps);
            barrier_init(low_empty + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 2 * kLate; ++i) {
            barrier_init(v_full + 8 * i, 4);
            barrier_init(v_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2 * kTiles; ++i) {
            barrier_init(s_full + 8 * i, 1);
            barrier_init(p_full + 8 * i, kTileRows);
        }
        barrier_init(q_full, kTiles * kTileRows);
        barrier_init(all_done, 1);
        for (int i = 0; i < kTiles; ++i) barrier_init(o_half + 8 * i, 1);
        barrier_fence();
        *dead = 0;
    }
    __syncthreads();
    if (start.limit == 0) return;
    const uint64_t u0 = start.flat;
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
    if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
        // ---- loader: a step's keys of both pages, then their values; page
        // numbers are looked up 32 blocks at a time
        Item it = start;
        uint32_t i = 0, g = 0;  // halves and steps so far
        bool ok = true;
        do {
            int page = -1;
            uint64_t shown = 0;
            const int n = it.to - it.from;
            for (int j = 0; j < n && ok; ++j, ++g) {
                if ((j & 15) == 0) {
                    const int block = it.lo + 2 * (it.from + j) + lane;
                    page = -1;
                    shown = 0;
                    if (block < it.hi && 2 * j + lane < 2 * n) {
                        page = __ldg(batch.page_table + static_cast<size_t>(it.seq) * batch.max_pages + block);
                        if (page < 0 || static_cast<uint32_t>(page) >= cache.n_pages) {
                            page = -1;
                            kv_invalid(batch);
                        } else {
                            shown = shown_tokens(p, it.seq, it.len, block);
                        }
                    }
                }
                for (int k = 0; k < 4; ++k, ++i) {
                    const uint32_t slot = i % kRaw;
                    const int from = __shfl_sync(kFull, page, (2 * j + (k & 1)) & 31);
                    const uint64_t bits = __shfl_sync(kFull, shown, (2 * j + (k & 1)) & 31);
                    ok = i < kRaw || wait(raw_empty + 8 * slot, i / kRaw - 1);
                    if (!ok) break;
                    if (lane == 0) {
                        if (k < 2) step_shown[(g & 7) * 2 + k] = bits;
                        if (from >= 0) {
                            barrier_expect(raw_full + 8 * slot, Cfg::kHalf);
                            bulk_load(shared_addr(smem + Cfg::kOffRaw + slot * Cfg::kHalf),
                                      cache.pages + ((static_cast<size_t>(from) * n_kv + it.head) * 2 + (k >> 1)) * Cfg::kHalf,
                                      Cfg::kHalf, raw_full + 8 * slot);
                        } else {
                            barrier_arrive(raw_full + 8 * slot);
                        }
                    }
                }
            }
        } while (ok && next_item(batch, p, n_kv, group, it));
        // copies in flight may not outlive the block's shared memory
        for (uint32_t k = i > kRaw ? i - kRaw : 0; k < i; ++k)
            if (!barrier_wait(raw_full + 8 * (k % kRaw), (k / kRaw) & 1)) *dead = 1;
    } else if (warp == kMmaWarp) {
        // ---- products, issued by one thread, page by page of a step: S of a
        // tile's page of the next step goes behind the product that reads this
        // step's P.  The tensor cores take one thread's products in order, so
        // S may be written where P was, and a commit behind S also stands for
        // the product before it.  At an item's end a commit without S does.
        // The whole warp runs this code and one elected lane issues: descriptors
        // are then warp-uniform values, which the instruction takes them as.
        Item it = start;
        const uint32_t base = shared_addr(smem);
        const uint64_t q_desc = operand_desc(base);
        const auto all_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(kFull, wait(bar, parity)) != 0; };
        // S of a tile at step g: the keys' upper parts, then the lower ones
        const auto scores = [&](int tile, uint32_t g) {
            const uint32_t late = g % kLate;
            const uint64_t q = q_desc + tile * (Cfg::kQTile >> 4);
            const uint64_t k = q_desc + (Cfg::kOffK >> 4) + (g & 1) * (Cfg::kKeys >> 4);
            const uint64_t low = q_desc + (Cfg::kOffLow >> 4) + late * (Cfg::kKeys >> 4);
            if (tile == 0) {
                if (!all_wait(k_full + 8 * (g & 1), g >> 1) || !all_wait(low_full + 8 * late, g / kLate)) return false;
                fence_after();
            }
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint64_t at = ((i / 4) * (kStepKeys * 128) + (i % 4) * 32) >> 4;
                    mma_shared_two(tmem + Cfg::kScores + tile * kStepKeys,
                                   q + (((i / 4) * (kTileRows * 128) + (i % 4) * 32) >> 4), k + at, low + at,
                                   mma_shape(kTileRows, kStepKeys), i > 0);
                }
                mma_commit(s_full + 16 * tile);
                mma_commit(s_full + 16 * tile + 8);
                if (tile == kTiles - 1) {
                    mma_commit(k_empty + 8 * (g & 1));
                    mma_commit(low_empty + 8 * late);
                }
            }
            return true;
        };
        const auto output = [&](int tile, int h, uint32_t g, uint32_t add) {
            const uint32_t late = g % kLate;
            const uint64_t v = q_desc + ((Cfg::kOffV + h * (D * 128)) >> 4) + late * (Cfg::kValues >> 4);
            if (tile == 0 && !all_wait(v_full + 16 * late + 8 * h, g / kLate)) return false;
            fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kKvPage / 16; ++k)
                    mma_tensor(tmem + Cfg::kOut + tile * D, tmem + Cfg::kScores + tile * kStepKeys + h * kKvPage + 8 * k,
                               v + (k * 32 >> 4), mma_shape(kTileRows, D), k > 0 ? 1u : add);
                if (h == 0) mma_commit(o_half + 8 * tile);
                if (tile == kTiles - 1) mma_commit(v_empty + 16 * late + 8 * h);
            }
            return true;
        };
        uint32_t g = 0, items = 0;  // steps and items so far
        bool ok = true;
        do {
            const int steps = __shfl_sync(kFull, it.to - it.from, 0);
            ok = all_wait(q_full, items);
            fence_after();
            for (int tile = 0; tile < kTiles; ++tile) ok = ok && scores(tile, g);
            for (int j = 0; j < steps && ok; ++j, ++g) {
                const bool more = j + 1 < steps;
#pragma unroll
                for (int i = 0; i < 2 * kTiles; ++i) {
                    const int tile = i % kTiles, h = i / kTiles;
                    ok = ok && all_wait(p_full + 16 * tile + 8 * h, g) && output(tile, h, g, j % kFold > 0 || h > 0);
                    if (!ok) break;
                    if (h == 0) continue;
                    if (more) {
                        ok = scores(tile, g + 1);
                    } else if (elect_one()) {
                        mma_commit(s_full + 16 * tile);
                        mma_commit(s_full + 16 * tile + 8);
                    }
                }
            }
            ++items;
        } while (ok && next_item(batch, p, n_kv, group, it));
        // nothing that was issued may outlive the block: a last commit stands
        // for all of it
        if (elect_one()) mma_commit(all_done);
        if (!barrier_wait(all_done, 0)) *dead = 1;
        __syncwarp();
    } else if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
        // ---- codes to f16 operands
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDecodeRegs));
        const int quarter = warp & 3;
        Item it = start;
        uint32_t g = 0;
        bool ok = true;
        if (warp < kSoftmaxWarps + kKeyWarps) {
            const int page = (warp - kSoftmaxWarps) >> 2;
            do {
                for (int j = it.from; j < it.to && ok; ++j, ++g) {
                    const uint32_t st = g & 1, late = g % kLate, turn = g / kLate - 1;  // turn: of the buffer's last use
                    const uint32_t i = 4 * g + page, slot = i % kRaw;
                    ok = wait(raw_full + 8 * slot, i / kRaw) && (g < 2 || wait(k_empty + 8 * st, (g >> 1) - 1));
                    if (!ok) break;
                    uint32_t high[KvChunk<D>::kGroups][2][8], low[KvChunk<D>::kGroups][2][8];
                    decode_keys<D>(smem + Cfg::kOffRaw + slot * Cfg::kHalf, quarter, high, low);
                    store_keys<D>(high, smem + Cfg::kOffK + st * Cfg::kKeys, page, quarter);
                    fence_shared();
                    __syncwarp();
                    if (lane == 0) {
                        barrier_arrive(k_full + 8 * st);
                        barrier_arrive(raw_empty + 8 * slot);
                    }
                    ok = g < kLate || wait(low_empty + 8 * late, turn);
                    if (!ok) break;
                    store_keys<D>(low, smem + Cfg::kOffLow + late * Cfg::kKeys, page, quarter);
                    fence_shared();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(low_full + 8 * late);
                }
            } while (ok && next_item(batch, p, n_kv, group, it));
        } else {
            do {
                for (int j = it.from; j < it.to && ok; ++j, ++g) {
                    const uint32_t late = g % kLate, turn = g / kLate - 1;
                    for (int page = 0; page < 2; ++page) {
                        const uint32_t i = 4 * g + 2 + page, slot = i % kRaw;
                        ok = wait(raw_full + 8 * slot, i / kRaw) && (g < kLate || wait(v_empty + 16 * late + 8 * page, turn));
                        if (!ok) break;
                        decode_values<D>(smem + Cfg::kOffRaw + slot * Cfg::kHalf,
                                         smem + Cfg::kOffV + late * Cfg::kValues + page * (D * 128), quarter,
                                         step_shown[(g & 7) * 2 + page]);
                        fence_shared();
                        __syncwarp();
                        if (lane == 0) {
                            barrier_arrive(v_full + 16 * late + 8 * page);
                            barrier_arrive(raw_empty + 8 * slot);
                        }
                    }
                }
            } while (ok && next_item(batch, p, n_kv, group, it));
        }
    } else if (warp < kSoftmaxWarps) {
        // ---- softmax: one thread a query column
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane, col = tile * kTileRows + row;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + Cfg::kScores + tile * kStepKeys, o_at = tmem + lanes + Cfg::kOut + tile * D;
        if (lane == 0) warp_items[warp] = start;
        __syncwarp();
        const Item& it = warp_items[warp];
        const auto advance = [&]() {
            Item next = it;
            __syncwarp();
            const bool more = next_item(batch, p, n_kv, group, next);
            if (lane == 0) warp_items[warp] = next;
            __syncwarp();
            return more;
        };
        uint32_t g = 0, sg = 0;  // steps, and commits of a page's S, so far
        bool ok = true;
        do {
            const bool on = col < it.cols;
            const int at_col = it.col0 + (on ? col : 0);
            int low, limit;
            row_limits(p, it.len - it.n_rows + at_col / group, it.len, low, limit);
            float unit = 1.0f;
            {
                const uint64_t src = static_cast<uint64_t>(it.first_row + at_col / group) * p.q_stride +
                                     static_cast<uint64_t>(it.head * group + at_col % group) * D;
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

            float ref = kNegInf;
            uint64_t l2 = 0;  // two parts of the sum of weights
            const int steps = it.to - it.from;
            int key0 = (it.lo + 2 * it.from) * kKvPage;
            for (int j = 0; j < steps && ok; ++j, ++g, ++sg) {
                for (int h = 0; h < 2; ++h, key0 += kKvPage) {
                    ok = wait(s_full + 16 * tile + 8 * h, sg);
                    if (!ok) break;
                    fence_after();
                    if (h == 0 && j > 0 && j % kFold == 0) fold_output<D>(o_at, parts, ref, unit, j == kFold);
                    const uint32_t sh = s_at + h * kKvPage;
                    const uint64_t shown = step_shown[(g & 7) * 2 + h];
                    if (shown != ~0ull || key0 + kKvPage - 1 > warp_limit || key0 <= warp_low) {
                        // hidden tokens' scores become -inf in place; the rest
                        // of the page's work then knows no mask
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            const int a = limit - (key0 + 32 * c), b = low - (key0 + 32 * c);
                            uint32_t see = static_cast<uint32_t>(shown >> (32 * c));
                            see &= a < 0 ? 0u : a >= 31 ? ~0u : (2u << a) - 1u;
                            see &= b < 0 ? ~0u : b >= 31 ? 0u : ~((2u << b) - 1u);
                            float v[32];
                            tensor_load(sh + 32 * c, v);
                            tensor_wait_load();
                            tensor_ready(v);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((see >> i) & 1)) v[i] = kNegInf;
                            tensor_store(sh + 32 * c, reinterpret_cast<const uint32_t*>(v));
                        }
                        tensor_wait_store();
                    }
                    // 32 tokens at a time, the next ones on their way
                    float v[2][32];
                    tensor_load(sh, v[0]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float(&x)[32] = v[c];
                        tensor_wait_load();
                        tensor_ready(x);
                        if (c == 0) tensor_load(sh + 32, v[1]);
                        // weights by the reference so far: their sum tells
                        // whether one may be too large for that
                        uint32_t w[16];
                        uint64_t sum = weigh(x, ref, unit, w);
                        const bool far = ref == kNegInf || !(first_of(sum) + second_of(sum) <= kMost);
                        if (__any_sync(kFull, far)) {
                            // the reference follows the maximum; what was
                            // weighed by the old one is rescaled
                            float f = 1.0f;
                            const float mx = largest(x);
                            if (far && mx > ref) {
                                f = ref == kNegInf ? 1.0f : exp2_fast((ref - mx) * unit);
                                ref = mx;
                            }
                            l2 = fma_two(l2, pair(f, f), 0);
                            if (c == 0) {
                                tensor_wait_load();
                                tensor_ready(v[1]);
                            } else {
                                tensor_wait_store();
                                scale_weights(sh, f);
                            }
                            if (h > 0 || j % kFold > 0) {
                                // behind the product of the page before
                                ok = h == 0 || wait(o_half + 8 * tile, g);
                                fence_after();
                                if (ok)
                                    for (int k = 0; k < D / 16; ++k) scale_output(o_at + 16 * k, f);
                            }
                            sum = weigh(x, ref, unit, w);
                        }
                        l2 = add_two(l2, sum);
                        // P takes the columns of S that have been read
                        tensor_store16(sh + 16 * c, w);
                    }
                    if (!ok) break;
                    tensor_wait_store();
                    fence_before();
                    barrier_arrive(p_full + 16 * tile + 8 * h);
                }
            }
            // ---- the output of this thread's column, or its partial result
            ok = ok && wait(s_full + 16 * tile, sg) && wait(s_full + 16 * tile + 8, sg);
            if (!ok) break;
            ++sg;
            fence_after();
            if (steps > kFold) unfold_output<D>(o_at, parts, ref, unit);
            const float l = first_of(l2) + second_of(l2), inv = l != 0.0f ? 1.0f / l : 0.0f;
            const float at = l != 0.0f ? fmaf(ref, unit, -kHead) : kNegInf;
            const uint64_t out_row = output_row(p, group, it.first_row, it.head, at_col);
            const bool whole = it.from == 0 && it.to == it.steps;
            float* part = parts + (2ull * blockIdx.x + (it.flat == u0 ? 0 : 1)) * kRowPartFloats<D>;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tensor_load(o_at + 32 * c, o);
                tensor_wait_load();
                tensor_ready(o);
                if (!on) continue;
                if (whole) {
                    uint16_t* out = static_cast<uint16_t*>(p.out) + out_row * D + 32 * c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        uint2 w = make_uint2(0u, 0u);
                        if (l != 0.0f)
                            w = make_uint2(kv_pack2(o[i] * inv, o[i + 1] * inv, p.dtype),
                                           kv_pack2(o[i + 2] * inv, o[i + 3] * inv, p.dtype));
                        *reinterpret_cast<uint2*>(out + i) = w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[(2 + 32 * c + i) * kWidth + col] = o[i];
                }
            }
            if (on && whole && p.lse) p.lse[out_row] = l != 0.0f ? (at + log2f(l)) * kLn2 : kNegInf;
            if (on && !whole) {
                part[col] = at;
                part[kWidth + col] = l;
            }
            fence_before();
        } while (advance());
    }

    __syncthreads();
    if (threadIdx.x == 0 && *dead) kv_timeout(batch);
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kColumns) : "memory");
    }
}

// Items that several blocks share: their partial results in block order, so
// that the sum does not depend on which block was done first.  Eight blocks an
// item, 32 columns each (38 MB of partial results of 147 blocks: 24 us).
constexpr int kJoinColumns = 32, kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_rows_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                    gofann_kv_attention_params p, uint32_t blocks,
                                                                    const float* __restrict__ parts)
{
    __shared__ float turn[kJoinColumns][D + 1];
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const uint32_t n_kv = cache.n_kv_heads;
    const uint64_t total = locate(batch, p, n_kv, group, ~0ull).total;
    const uint64_t share = steps_per_block(total, blocks);
    // block i joins the item that the end of share i cuts, if that is the item's first cut
    const uint64_t cut = share * (blockIdx.y + 1);
    if (cut >= total) {
        wait_previous();
        return;
    }
    const Place at = locate(batch, p, n_kv, group, cut);
    Item it{};
    it.seq = at.seq, it.head = at.head, it.tile = at.tile, it.flat = cut, it.limit = ~0ull;
    open_item(batch, p, group, at.step, it);
    const uint64_t begin = cut - at.step, end = begin + it.steps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = static_cast<int>(blockIdx.x) * kJoinColumns;
    wait_previous();
    if (begin >= cut || begin < share * blockIdx.y || c0 >= it.cols) return;
    const uint64_t last = (end - 1) / share;
    constexpr int kEach = D / (kJoinThreads / 32);
    float m = kNegInf, l = 0.0f, o[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) o[k] = 0.0f;
    if (c0 + lane < it.cols) {
        for (uint64_t b = blockIdx.y; b <= last; ++b) {
            const float* part = parts + (2 * b + (begin <= share * b ? 0 : 1)) * kRowPartFloats<D> + c0 + lane;
            const float pm = __ldcg(part), pl = __ldcg(part + kWidth);
            const float top = fmaxf(m, pm), base = top == kNegInf ? 0.0f : top;
            const float f = exp2_fast(m - base), h = exp2_fast(pm - base);
            l = l * f + pl * h;
#pragma unroll
            for (int k = 0; k < kEach; ++k) o[k] = o[k] * f + __ldcg(part + (2 + warp * kEach + k) * kWidth) * h;
            m = top;
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) turn[lane][warp * kEach + k] = l != 0.0f ? o[k] * inv : 0.0f;
    if (warp == 0 && p.lse && c0 + lane < it.cols)
        p.lse[output_row(p, group, it.first_row, it.head, it.col0 + c0 + lane)] = l != 0.0f ? (m + log2f(l)) * kLn2 : kNegInf;
    __syncthreads();
    for (int i = threadIdx.x; i < kJoinColumns * (D / 2); i += kJoinThreads) {
        const int c = i / (D / 2), d = i % (D / 2) * 2;
        if (c0 + c >= it.cols) break;
        const uint64_t row = output_row(p, group, it.first_row, it.head, it.col0 + c0 + c);
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row * D + d) =
            kv_pack2(turn[c][d], turn[c][d + 1], p.dtype);
    }
}

// One thread block per SM, no more than there can be items of one step.
uint32_t row_blocks(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p)
{
    const uint64_t cols = static_cast<uint64_t>(batch.n_rows) * (p.n_heads / cache.n_kv_heads);
    const uint64_t most = (cols / kWidth + batch.n_seqs) * cache.n_kv_heads * (batch.max_pages / 2 + 1ull);
    const int sms = sm_count();
    const uint64_t want = sms > 0 ? sms : 1;
    return static_cast<uint32_t>(most < want ? most : want);
}

template <int D>
int launch_rows(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                float* parts, cudaStream_t s)
{
    auto* kernel = kv_attend_rows_kernel<D>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Rows<D>::kBytes);
    if (e != cudaSuccess) return cuda_status(e, "kv_attention: shared memory attribute");
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && (p.q_stride & 3) == 0;
    const uint32_t blocks = row_blocks(cache, batch, p);
    kernel<<<blocks, kRowThreads, Rows<D>::kBytes, s>>>(cache, batch, p, wide, parts);
    GOFANN_CHECK_LAUNCH("kv_attend_rows_kernel");
    if (blocks == 1) return GOFANN_OK;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kWidth / kJoinColumns, blocks - 1);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv_join_rows_kernel<D>, cache, batch, p, blocks, static_cast<const float*>(parts));
    if (e != cudaSuccess) return cuda_status(e, "kv_join_rows_kernel");
    return GOFANN_OK;
}

}  // namespace

size_t attend_rows_scratch(uint32_t head_dim, int sms)
{
    return 3 * sizeof(float) * (head_dim == 64 ? kRowPartFloats<64> : kRowPartFloats<128>) * static_cast<size_t>(sms);
}

int attend_rows(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                float* parts, cudaStream_t s)
{
    return cache.head_dim == 64 ? launch_rows<64>(cache, batch, p, parts, s)
                                : launch_rows<128>(cache, batch, p, parts, s);
}

}  // namespace gofann
