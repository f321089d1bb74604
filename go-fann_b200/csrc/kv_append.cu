// kv_append.cu — rotary positions, 4-bit quantisation into the paged cache
// and the 8-bit bounds of the touched blocks, in one launch.
//
// One block owns one (touched page, key/value head): it rotates the query
// heads of its head's group and the keys of the page's new tokens, quantises
// keys and values into shared memory, merges the codes into the page's words
// and renews the page's bounds from all tokens it holds.  Two tokens share
// code bytes and words, so a single owner is what makes the merge safe.
#include "kv_common.cuh"

namespace gofann {

int kv_check(const char* who, const gofann_kv_cache* cache, const gofann_kv_batch* batch, int dtype, uint32_t n_heads)
{
    if (!cache || !batch) return fail(GOFANN_ERR_INVALID, "%s: null descriptor", who);
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return fail(GOFANN_ERR_UNSUPPORTED, "%s: head_dim %u (64 or 128)", who, cache->head_dim);
    if (dtype != GOFANN_DTYPE_BF16 && dtype != GOFANN_DTYPE_F16)
        return fail(GOFANN_ERR_INVALID, "%s: dtype %d (GOFANN_DTYPE_BF16 or GOFANN_DTYPE_F16)", who, dtype);
    if (cache->n_kv_heads == 0 || n_heads == 0 || n_heads % cache->n_kv_heads != 0)
        return fail(GOFANN_ERR_INVALID, "%s: %u query heads over %u key/value heads (a positive multiple)", who, n_heads,
                    cache->n_kv_heads);
    if (n_heads > 65535u) return fail(GOFANN_ERR_UNSUPPORTED, "%s: %u query heads (at most 65535)", who, n_heads);
    if (cache->n_pages > 0x7fffffffu)
        return fail(GOFANN_ERR_UNSUPPORTED, "%s: %u pages (at most 2^31 - 1)", who, cache->n_pages);
    if (batch->max_pages > (1u << 24))
        return fail(GOFANN_ERR_UNSUPPORTED, "%s: %u pages per sequence (at most 2^24)", who, batch->max_pages);
    if (batch->n_rows > (1u << 24) || batch->n_seqs > (1u << 24))
        return fail(GOFANN_ERR_UNSUPPORTED, "%s: %u rows of %u sequences (at most 2^24)", who, batch->n_rows, batch->n_seqs);
    if (batch->n_rows && (!batch->seq_len || !batch->row_offset || batch->n_seqs == 0))
        return fail(GOFANN_ERR_INVALID, "%s: rows without sequences", who);
    if (batch->n_rows && batch->max_pages && !batch->page_table)
        return fail(GOFANN_ERR_INVALID, "%s: null page table", who);
    return GOFANN_OK;
}

namespace {

// Pages that sequence s's rows touch.
__device__ __forceinline__ uint32_t touched_pages(const gofann_kv_batch& b, uint32_t s)
{
    int first, n;
    kv_rows(b, s, first, n);
    const int len = kv_len(b, s);
    if (n == 0 || len == 0) return 0;
    const int start = len > n ? len - n : 0;
    return static_cast<uint32_t>((len + kKvPage - 1) / kKvPage - start / kKvPage);
}

template <bool kBf16>
__device__ __forceinline__ uint4 pack8(const float (&x)[8])
{
    constexpr int t = kBf16 ? GOFANN_DTYPE_BF16 : GOFANN_DTYPE_F16;
    return make_uint4(kv_pack2(x[0], x[1], t), kv_pack2(x[2], x[3], t), kv_pack2(x[4], x[5], t), kv_pack2(x[6], x[7], t));
}

// How a call's rows are rotated.  Half and Pairs: whole lanes of eight
// dimensions are rotated or not; Any: every other form, through shared memory.
enum { kRotateNone, kRotateHalf, kRotatePairs, kRotateAny };

// cos and sin of this lane's eight dimensions; sin with the sign that it has
// in x_a cos - x_b sin, x_b cos + x_a sin.
template <int kMode>
__device__ __forceinline__ void load_angles(const gofann_kv_append_params& p, int pos, int d0, float (&c)[8], float (&s)[8])
{
    const int rotary = static_cast<int>(p.rotary_dim), half = rotary >> 1;
    const size_t row = static_cast<size_t>(pos) * half;
    if (kMode == kRotateHalf) {
        if (d0 >= rotary) return;
        const bool low = d0 < half;
        const int i = low ? d0 : d0 - half;
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos + row + i + k));
            const float4 b = __ldg(reinterpret_cast<const float4*>(p.sin + row + i + k));
            c[k] = a.x, c[k + 1] = a.y, c[k + 2] = a.z, c[k + 3] = a.w;
            s[k] = low ? -b.x : b.x, s[k + 1] = low ? -b.y : b.y, s[k + 2] = low ? -b.z : b.z, s[k + 3] = low ? -b.w : b.w;
        }
    } else if (kMode == kRotatePairs) {
        if (d0 >= rotary) return;
        const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos + row + d0 / 2));
        const float4 b = __ldg(reinterpret_cast<const float4*>(p.sin + row + d0 / 2));
        c[0] = c[1] = a.x, c[2] = c[3] = a.y, c[4] = c[5] = a.z, c[6] = c[7] = a.w;
        s[0] = -b.x, s[1] = b.x, s[2] = -b.y, s[3] = b.y, s[4] = -b.z, s[5] = b.z, s[6] = -b.w, s[7] = b.w;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int d = d0 + k;
            if (d >= rotary) continue;
            const bool low = p.interleaved ? (d & 1) == 0 : d < half;
            const int i = p.interleaved ? d >> 1 : (d < half ? d : d - half);
            c[k] = __ldg(p.cos + row + i);
            const float b = __ldg(p.sin + row + i);
            s[k] = low ? -b : b;
        }
    }
}

// Rotates this lane's eight dimensions of a vector that consecutive lanes
// hold; every product and sum rounded by itself.  All lanes of the warp call
// it.
template <int kMode, bool kBf16>
__device__ __forceinline__ void rotate8(const gofann_kv_append_params& p, const uint4& raw, int d0, const float (&c)[8],
                                        const float (&s)[8], float* stage, float (&x)[8])
{
    const int rotary = static_cast<int>(p.rotary_dim), half = rotary >> 1;
    float o[8];  // the other element of each pair
    if (kMode == kRotateHalf) {
        const int lane = threadIdx.x & 31, src = d0 >= rotary ? lane : d0 < half ? lane + half / 8 : lane - half / 8;
        uint4 w;
        w.x = __shfl_sync(kFull, raw.x, src);
        w.y = __shfl_sync(kFull, raw.y, src);
        w.z = __shfl_sync(kFull, raw.z, src);
        w.w = __shfl_sync(kFull, raw.w, src);
        unpack8<kBf16>(w, o);
    } else if (kMode == kRotatePairs) {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = x[k ^ 1];
    } else {
        __syncwarp();
        *reinterpret_cast<float4*>(stage + d0) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(stage + d0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int d = d0 + k;
            o[k] = d < rotary ? stage[p.interleaved ? d ^ 1 : d < half ? d + half : d - half] : 0.0f;
        }
    }
    if (kMode != kRotateAny && d0 >= rotary) return;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (kMode != kRotateAny || d0 + k < rotary) x[k] = __fadd_rn(__fmul_rn(x[k], c[k]), __fmul_rn(o[k], s[k]));
}

// Eight values of a group that eight lanes hold: their codes, the values that
// those stand for and the group's params (f16 scale below, minimum above).
// All lanes of the warp call it.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], float (&code)[8])
{
    float mn, mx;
    const auto range = [&]() {
        mn = mx = x[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) {
            mn = fminf(mn, x[k]);
            mx = fmaxf(mx, x[k]);
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
            mn = fminf(mn, __shfl_xor_sync(kFull, mn, off));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, off));
        }
    };
    range();
    bool bad = mn < -GOFANN_KV_CLAMP || mx > GOFANN_KV_CLAMP;
#pragma unroll
    for (int k = 0; k < 8; ++k) bad |= x[k] != x[k];
    if (__any_sync(kFull, bad)) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            x[k] = x[k] == x[k] ? fminf(fmaxf(x[k], -GOFANN_KV_CLAMP), GOFANN_KV_CLAMP) : 0.0f;
        range();
    }
    const __half hs = __float2half_rn(__fdiv_rn(__fsub_rn(mx, mn), 15.0f)), hm = __float2half_rn(mn);
    const float scale = __half2float(hs), m = __half2float(hm);
    // rint of the quotient: by the reciprocal (off by less than 3e-6 below 16),
    // unless that is so near a half that the rounded quotient might fall to
    // the other side
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    bool near = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float t = __fmul_rn(__fsub_rn(x[k], m), inv);
        code[k] = rintf(t);
        near |= fabsf(t - code[k]) > 0.49998f;
    }
    if (near) {
#pragma unroll
        for (int k = 0; k < 8; ++k) code[k] = scale > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x[k], m), scale)) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        code[k] = fminf(fmaxf(code[k], 0.0f), 15.0f);
        x[k] = __fadd_rn(__fmul_rn(code[k], scale), m);
    }
    return static_cast<uint32_t>(__half_as_ushort(hs)) | (static_cast<uint32_t>(__half_as_ushort(hm)) << 16);
}

// Eight codes of a token that the page holds, from dimension d0 on, the values
// of a key's and the params of their group.
template <int D>
__device__ __forceinline__ uint32_t held_key(const uint8_t* chunk, int token, int d0, float (&x)[8], float (&code)[8])
{
    const int g = 2 * (token >> 4) + (token & 1), kt = (token >> 2) & 3, r = (token >> 1) & 1, grp = d0 / kKvGroup;
    const uint32_t sm = reinterpret_cast<const uint32_t*>(chunk + KvChunk<D>::kKeyParams)[kv_param_word<D>(token) + grp];
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffff)));
    const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int d = d0 + k, tj = (d >> 2) & 15, n = (d >> 1) & 1, e = d & 1;
        code[k] = static_cast<float>((chunk[(((kt * KvChunk<D>::kGroups + grp) * 8 + g) * 16 + tj) * 4 + 2 * e + r] >> (4 * n)) & 15);
        x[k] = __fadd_rn(__fmul_rn(code[k], s), m);
    }
    return sm;
}
template <int D>
__device__ __forceinline__ uint32_t held_value(const uint8_t* chunk, int token, int d0, float (&code)[8])
{
    const int t = token >> 4, kt = (token >> 2) & 3, n = (token >> 1) & 1, e = token & 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int d = d0 + k, dt = d >> 4, r = (d >> 3) & 1, g = d & 7;
        code[k] = static_cast<float>((chunk[KvChunk<D>::kValueCodes + (((dt * 8 + g) * 4 + t) * 4 + kt) * 4 + 2 * e + r] >> (4 * n)) & 15);
    }
    return reinterpret_cast<const uint32_t*>(chunk + KvChunk<D>::kValueParams)[kv_param_word<D>(token) + d0 / kKvGroup];
}

// The page words [i] of this thread, and the nibbles of them that the rows
// [lo, hi) of the page write.
__device__ __forceinline__ uint32_t key_mask(int i, int G, int lo, int hi)
{
    const int g = (i >> 4) & 7, kt = (i >> 7) / G, k0 = 16 * (g >> 1) + 4 * kt + (g & 1);
    return (k0 >= lo && k0 < hi ? 0x00ff00ffu : 0u) | (k0 + 2 >= lo && k0 + 2 < hi ? 0xff00ff00u : 0u);
}
__device__ __forceinline__ uint32_t value_mask(int i, int lo, int hi)
{
    const int k1 = 16 * ((i >> 2) & 3) + 4 * (i & 3);  // tokens k1 .. k1 + 3: 2 n + e
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (k1 + q >= lo && k1 + q < hi) m |= 0x0f0fu << (16 * (q & 1) + 4 * (q >> 1));
    return m;
}

// What bounds it: a full page is a stream (q, k, v in, q, k, v out, codes),
// a decode step's single rows are the chain of dependent loads: sequence, page
// number, then everything else at once (one row 8.5 us, 96 rows 10.7 us).  Five
// chunks of 2043 rows (32 query and 8 key/value heads of 64, in pairs) take 45
// us, 2.9 TB/s: 28 M instructions of a warp, 56 % of the issue slots, half of
// them rounding and rotating; the rest is the wait for a page's first rows.  So all that a block reads is asked
// for before it is used: page words that are only partly written, the keys
// that the page holds, the rows.
template <int D, int kMode, bool kBf16, int kAppendThreads>
__global__ void __launch_bounds__(kAppendThreads, kAppendThreads == 128 ? 4 : 3) kv_append_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                   gofann_kv_append_params p, bool q_wide,
                                                                   bool kv_wide)
{
    using Chunk = KvChunk<D>;
    constexpr int G = Chunk::kGroups;
    constexpr int kLanes = D / 8;                           // lanes of one vector
    constexpr int kVectors = kAppendThreads / kLanes;       // vectors at a time
    constexpr int kWords = Chunk::kCodes / 4 / kAppendThreads;  // of keys (and of values) per thread
    constexpr int kParts = kAppendThreads / (16 * G);       // threads that share four dimensions of the old keys
    constexpr int kKeyRow = D == 128 ? 192 : 64;            // bytes: rows of two tokens in different banks
    constexpr int kValueRow = kKvPage + 4;
    __shared__ __align__(16) uint8_t key_codes[kKvPage * kKeyRow];  // [token][dim]
    __shared__ __align__(16) uint8_t value_codes[D * kValueRow];    // [dim][token]
    __shared__ uint32_t params[2][kKvPage][G];
    __shared__ __align__(16) float high_of[kVectors + kParts][D], low_of[kVectors + kParts][D];
    __shared__ float top[kAppendThreads / 32];
    __shared__ int missing;  // whether a row has no position in the tables

    const uint32_t head = blockIdx.y;
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && head == 0 && batch.status) {
        kv_check_sequences(batch, threadIdx.x, kAppendThreads);
        for (uint32_t s = threadIdx.x; s < batch.n_seqs; s += kAppendThreads) {
            int first, n;
            kv_rows(batch, s, first, n);
            if (n > kv_len(batch, s)) kv_invalid(batch);  // rows before the sequence's first token
        }
    }
    if (kMode != kRotateNone) {
        if (threadIdx.x == 0) missing = 0;  // (a flag in registers: chunks of 2043 rows 47 us instead of 45)
        __syncthreads();
    }
    uint32_t seq, at;
    if (!kv_find(batch.n_seqs, blockIdx.x, [&](uint32_t s) { return touched_pages(batch, s); }, seq, at)) return;
    int first_row, n_rows;
    kv_rows(batch, seq, first_row, n_rows);
    const int len = kv_len(batch, seq);
    const int start = len - n_rows;  // position of the first row; negative where rows exceed the length
    const int block = (start > 0 ? start / kKvPage : 0) + static_cast<int>(at);
    const int base = block * kKvPage;
    const int lo = start > base ? start - base : 0;              // first new token of the page
    const int hi = len - base < kKvPage ? len - base : kKvPage;  // tokens that the page holds
    const int32_t page = __ldg(batch.page_table + static_cast<size_t>(seq) * batch.max_pages + block);
    const bool page_ok = page >= 0 && static_cast<uint32_t>(page) < cache.n_pages;
    if (!page_ok && threadIdx.x == 0) kv_invalid(batch);
    uint8_t* chunk = cache.pages + (static_cast<size_t>(page_ok ? page : 0) * cache.n_kv_heads + head) * Chunk::kBytes;
    uint32_t* kw = reinterpret_cast<uint32_t*>(chunk);
    uint32_t* vw = reinterpret_cast<uint32_t*>(chunk + Chunk::kValueCodes);
    uint32_t* kp = reinterpret_cast<uint32_t*>(chunk + Chunk::kKeyParams);
    uint32_t* vp = reinterpret_cast<uint32_t*>(chunk + Chunk::kValueParams);

    // ---- words that keep some of their nibbles
    uint32_t old_k[kWords], old_v[kWords];
#pragma unroll
    for (int n = 0; n < kWords; ++n) {
        const int i = threadIdx.x + n * kAppendThreads;
        const uint32_t mk = key_mask(i, G, lo, hi), mv = value_mask(i, lo, hi);
        old_k[n] = page_ok && mk && mk != ~0u ? kw[i] : 0u;
        old_v[n] = page_ok && mv && mv != ~0u ? vw[i] : 0u;
    }
    // ---- largest and smallest of the keys that the page held before: four
    // dimensions a thread, of every kParts-th pair of tokens
    if (cache.bounds) {
        const int combo = threadIdx.x % (16 * G), part = threadIdx.x / (16 * G);
        const int grp = combo / 16, tj = combo % 16;
        float h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = kNegInf, l[k] = -kNegInf;
        if (lo > 0 && page_ok) {
#pragma unroll
            for (int n = 0; n < 32 / kParts; ++n) {
                const int pairs = part + n * kParts, g = pairs & 7, kt = pairs >> 3;
                const int token = 16 * (g >> 1) + 4 * kt + (g & 1);
                if (token >= lo) continue;
                const uint32_t w = kw[((kt * G + grp) * 8 + g) * 16 + tj];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (token + 2 * r >= lo) continue;
                    const uint32_t sm = kp[((g * 4 + kt) * 2 + r) * G + grp], b = w >> (8 * r);
                    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffff)));
                    const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
                    const uint32_t c[4] = {b & 0xf, (b >> 16) & 0xf, (b >> 4) & 0xf, (b >> 20) & 0xf};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x = __fadd_rn(__fmul_rn(static_cast<float>(c[k]), s), m);
                        h[k] = fmaxf(h[k], x);
                        l[k] = fminf(l[k], x);
                    }
                }
            }
        }
        const int d = 64 * grp + 4 * tj;  // dimension 64 grp + 16 t + 4 j
        *reinterpret_cast<float4*>(&high_of[kVectors + part][d]) = make_float4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<float4*>(&low_of[kVectors + part][d]) = make_float4(l[0], l[1], l[2], l[3]);
    }

    // ---- rotate and quantise: a group of lanes takes a token, its query
    // heads, its key and its value; where there are fewer tokens than groups,
    // several groups share a token's query heads
    const uint32_t group = p.n_heads / cache.n_kv_heads;
    const int n_q = p.q ? static_cast<int>(group) : 0, tokens = hi - lo;
    const int vec = threadIdx.x / kLanes, d0 = (threadIdx.x % kLanes) * 8;
    const int share = tokens < kVectors ? kVectors / tokens : 1;  // groups of a token
    const int part = share > 1 ? vec / tokens : 0;
    const int step = share > 1 ? tokens : kVectors, turns = (n_q + share - 1) / share;
    float high[8], low[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) high[k] = kNegInf, low[k] = -kNegInf;
    for (int t0 = 0; t0 < tokens; t0 += step) {
        const int token = lo + t0 + (share > 1 ? vec % tokens : vec);
        const bool on = token < hi && part < share;
        const int row = first_row + base + (on ? token : lo) - start;
        const uint4 raw_k = load8(p.k, static_cast<uint64_t>(row) * p.k_stride + head * D + d0, kv_wide);
        const uint4 raw_v = load8(p.v, static_cast<uint64_t>(row) * p.v_stride + head * D + d0, kv_wide);
        const uint64_t q_at = static_cast<uint64_t>(row) * p.q_stride + head * group * D + d0;
        const auto fetch = [&](int kind) {
            return kind < n_q ? load8(p.q, q_at + static_cast<uint64_t>(kind) * D, q_wide) : make_uint4(0u, 0u, 0u, 0u);
        };
        // query vectors on their way: chunks of 2043 rows 51 us with 2, 45 with 4, 47 with 6
        constexpr int kAhead = 4;
        uint4 next[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) next[a] = fetch(part + a * share);
        float c[8], s[8];
        bool write = on;  // not where the tables have no such position
        if (kMode != kRotateNone) {
            int pos = p.positions ? __ldg(p.positions + row) : base + (on ? token : lo);
            if (pos < 0 || static_cast<uint32_t>(pos) >= p.n_positions) {
                if (d0 == 0) missing = 1;
                write = false;
                pos = 0;
            }
            load_angles<kMode>(p, pos, d0, c, s);
        }
        uint16_t* q_out = static_cast<uint16_t*>(p.q_out) + (static_cast<uint64_t>(row) * p.n_heads + head * group) * D + d0;
        for (int turn = 0; turn < turns; ++turn) {
            const int kind = part + turn * share;
            const uint4 raw = next[0];
#pragma unroll
            for (int a = 0; a + 1 < kAhead; ++a) next[a] = next[a + 1];
            next[kAhead - 1] = fetch(kind + kAhead * share);
            float x[8];
            unpack8<kBf16>(raw, x);
            if (kMode != kRotateNone) rotate8<kMode, kBf16>(p, raw, d0, c, s, low_of[vec], x);
            if (write && kind < n_q) *reinterpret_cast<uint4*>(q_out + kind * D) = pack8<kBf16>(x);
        }
        float x[8], code[8];
        unpack8<kBf16>(raw_k, x);
        // (low_of's row is free until the bounds are written)
        if (kMode != kRotateNone) rotate8<kMode, kBf16>(p, raw_k, d0, c, s, low_of[vec], x);
        const uint32_t kp_word = quantise8(x, code);
        const uint64_t kv_out = (static_cast<uint64_t>(row) * cache.n_kv_heads + head) * D + d0;
        const bool mine = write && part == 0;
        if (mine) {
            uint32_t c8[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                c8[k >> 2] |= static_cast<uint32_t>(code[k]) << (8 * (k & 3));
                high[k] = fmaxf(high[k], x[k]);
                low[k] = fminf(low[k], x[k]);
            }
            *reinterpret_cast<uint2*>(&key_codes[token * kKeyRow + d0]) = make_uint2(c8[0], c8[1]);
            if ((d0 & (kKvGroup - 1)) == 0) params[0][token][d0 / kKvGroup] = kp_word;
            if (p.k_out) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k_out) + kv_out) = pack8<kBf16>(x);
        }
        unpack8<kBf16>(raw_v, x);
        const uint32_t vp_word = quantise8(x, code);
        if (mine) {
#pragma unroll
            for (int k = 0; k < 8; ++k) value_codes[(d0 + k) * kValueRow + token] = static_cast<uint8_t>(code[k]);
            if ((d0 & (kKvGroup - 1)) == 0) params[1][token][d0 / kKvGroup] = vp_word;
            if (p.v_out) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v_out) + kv_out) = pack8<kBf16>(x);
        }
    }
    if (!page_ok) return;
    if (kMode == kRotateAny) __syncwarp();  // the stage was low_of's row
    if (cache.bounds) {
        *reinterpret_cast<float4*>(&high_of[vec][d0]) = make_float4(high[0], high[1], high[2], high[3]);
        *reinterpret_cast<float4*>(&high_of[vec][d0 + 4]) = make_float4(high[4], high[5], high[6], high[7]);
        *reinterpret_cast<float4*>(&low_of[vec][d0]) = make_float4(low[0], low[1], low[2], low[3]);
        *reinterpret_cast<float4*>(&low_of[vec][d0 + 4]) = make_float4(low[4], low[5], low[6], low[7]);
    }
    __syncthreads();
    if (kMode != kRotateNone && missing) {
        if (threadIdx.x == 0) kv_invalid(batch);
        // rows that are not written: their places keep the tokens that they hold
        for (int token = lo + vec; token < hi; token += kVectors) {
            const int pos = p.positions ? __ldg(p.positions + first_row + base + token - start) : base + token;
            if (pos >= 0 && static_cast<uint32_t>(pos) < p.n_positions) continue;
            float x[8], code[8];
            params[0][token][d0 / kKvGroup] = held_key<D>(chunk, token, d0, x, code);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                key_codes[token * kKeyRow + d0 + k] = static_cast<uint8_t>(code[k]);
                high_of[vec][d0 + k] = fmaxf(high_of[vec][d0 + k], x[k]);
                low_of[vec][d0 + k] = fminf(low_of[vec][d0 + k], x[k]);
            }
            params[1][token][d0 / kKvGroup] = held_value<D>(chunk, token, d0, code);
#pragma unroll
            for (int k = 0; k < 8; ++k) value_codes[(d0 + k) * kValueRow + token] = static_cast<uint8_t>(code[k]);
        }
        __syncthreads();
    }

    // ---- merge the codes into the page's words
#pragma unroll
    for (int n = 0; n < kWords; ++n) {
        const int i = threadIdx.x + n * kAppendThreads;
        const uint32_t mk = key_mask(i, G, lo, hi), mv = value_mask(i, lo, hi);
        if (mk) {
            // key word [kt][grp][g][t][j]: tokens k0 (even bytes) and k0 + 2, dimensions d .. d + 3
            const int j = i & 3, t = (i >> 2) & 3, g = (i >> 4) & 7, grp = (i >> 7) % G, kt = (i >> 7) / G;
            const int k0 = 16 * (g >> 1) + 4 * kt + (g & 1), d = 64 * grp + 16 * t + 4 * j;
            uint32_t word = 0;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(&key_codes[(k0 + 2 * r) * kKeyRow + d]);
                word |= ((c & 0xf) | ((c >> 12) & 0xf0) | ((c << 8) & 0x000f0000) | ((c >> 4) & 0x00f00000)) << (8 * r);
            }
            kw[i] = (word & mk) | (old_k[n] & ~mk);
        }
        if (mv) {
            // value word [dt][g][t][kt]: dimensions dv and dv + 8, tokens k1 .. k1 + 3 = 2 n + e: nibble n of bytes 2 e + r
            const int vkt = i & 3, vt = (i >> 2) & 3, vg = (i >> 4) & 7, dt = i >> 7;
            const int k1 = 16 * vt + 4 * vkt, dv = 16 * dt + vg;
            uint32_t word = 0;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(&value_codes[(dv + 8 * r) * kValueRow + k1]);
                word |= ((c & 0xf) | ((c >> 12) & 0xf0) | ((c << 8) & 0x000f0000) | ((c >> 4) & 0x00f00000)) << (8 * r);
            }
            vw[i] = (word & mv) | (old_v[n] & ~mv);
        }
    }
    for (int i = threadIdx.x; i < tokens * G; i += kAppendThreads) {
        const int token = lo + i / G, grp = i % G, w = kv_param_word<D>(token) + grp;
        kp[w] = params[0][token][grp];
        vp[w] = params[1][token][grp];
    }

    // ---- bounds of the page's tokens: a thread a dimension
    if (!cache.bounds) return;
    float h = kNegInf, l = -kNegInf;
    if (threadIdx.x < D) {
#pragma unroll
        for (int v = 0; v < kVectors + kParts; ++v) {
            h = fmaxf(h, high_of[v][threadIdx.x]);
            l = fminf(l, low_of[v][threadIdx.x]);
        }
    }
    float a = threadIdx.x < D ? fmaxf(fabsf(h), fabsf(l)) : 0.0f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(kFull, a, off));
    if (lane == 0) top[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x >= D) return;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) a = fmaxf(a, top[w]);
    const float scale = __fdiv_rn(a, 127.0f);
    const size_t entry = static_cast<size_t>(page) * cache.n_kv_heads + head;
    float h8 = 0.0f, l8 = 0.0f;
    if (scale > 0.0f) {
        h8 = fminf(fmaxf(ceilf(__fdiv_rn(h, scale)), -127.0f), 127.0f);
        l8 = fminf(fmaxf(floorf(__fdiv_rn(l, scale)), -127.0f), 127.0f);
    }
    int8_t* bounds = cache.bounds + entry * 2 * D;
    bounds[threadIdx.x] = static_cast<int8_t>(h8);
    bounds[D + threadIdx.x] = static_cast<int8_t>(l8);
    if (threadIdx.x == 0) cache.bound_scale[entry] = scale;
}

template <int D, int kMode, bool kBf16>
void launch_typed(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_append_params& p,
                  bool q_wide, bool kv_wide, dim3 grid, cudaStream_t s)
{
    // Blocks with a few rows wait for memory most of their time: small ones, so
    // that more of them fit an SM (96 sequences of one row, 4 heads: 11 us
    // instead of 14; for 8 blocks there is no difference).
    if (batch.max_rows <= 8)
        kv_append_kernel<D, kMode, kBf16, 128><<<grid, 128, 0, s>>>(cache, batch, p, q_wide, kv_wide);
    else
        kv_append_kernel<D, kMode, kBf16, 256><<<grid, 256, 0, s>>>(cache, batch, p, q_wide, kv_wide);
}
template <int D, int kMode>
void launch_mode(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_append_params& p,
                 bool q_wide, bool kv_wide, dim3 grid, cudaStream_t s)
{
    if (p.dtype == GOFANN_DTYPE_BF16)
        launch_typed<D, kMode, true>(cache, batch, p, q_wide, kv_wide, grid, s);
    else
        launch_typed<D, kMode, false>(cache, batch, p, q_wide, kv_wide, grid, s);
}
template <int D>
void launch_append(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_append_params& p, int mode,
                   bool q_wide, bool kv_wide, dim3 grid, cudaStream_t s)
{
    if (mode == kRotateNone)
        launch_mode<D, kRotateNone>(cache, batch, p, q_wide, kv_wide, grid, s);
    else if (mode == kRotateHalf)
        launch_mode<D, kRotateHalf>(cache, batch, p, q_wide, kv_wide, grid, s);
    else if (mode == kRotatePairs)
        launch_mode<D, kRotatePairs>(cache, batch, p, q_wide, kv_wide, grid, s);
    else
        launch_mode<D, kRotateAny>(cache, batch, p, q_wide, kv_wide, grid, s);
}

}  // namespace
}  // namespace gofann

using namespace gofann;

extern "C" {

size_t gofann_kv_chunk_bytes(uint32_t head_dim)
{
    return head_dim == 64 ? KvChunk<64>::kBytes : head_dim == 128 ? KvChunk<128>::kBytes : 0;
}

int gofann_kv_append(const gofann_kv_cache* cache, const gofann_kv_batch* batch, const gofann_kv_append_params* params,
                     void* stream)
{
    if (!params) return fail(GOFANN_ERR_INVALID, "kv_append: null descriptor");
    const gofann_kv_append_params& p = *params;
    int st = kv_check("kv_append", cache, batch, p.dtype, p.n_heads);
    if (st != GOFANN_OK) return st;
    const uint32_t d = cache->head_dim;
    if (p.rotary_dim > d || (p.rotary_dim & 1))
        return fail(GOFANN_ERR_INVALID, "kv_append: rotary_dim %u (even, at most head_dim %u)", p.rotary_dim, d);
    if (batch->n_rows == 0) return GOFANN_OK;
    if (!cache->pages || !p.k || !p.v) return fail(GOFANN_ERR_INVALID, "kv_append: null pages, keys or values");
    if ((p.q == nullptr) != (p.q_out == nullptr)) return fail(GOFANN_ERR_INVALID, "kv_append: q and q_out go together");
    if ((cache->bounds == nullptr) != (cache->bound_scale == nullptr))
        return fail(GOFANN_ERR_INVALID, "kv_append: bounds and bound_scale go together");
    if (p.rotary_dim && (!p.cos || !p.sin || p.n_positions == 0))
        return fail(GOFANN_ERR_INVALID, "kv_append: rotary_dim %u without tables", p.rotary_dim);
    if ((p.q && p.q_stride < static_cast<uint64_t>(p.n_heads) * d) ||
        p.k_stride < static_cast<uint64_t>(cache->n_kv_heads) * d || p.v_stride < static_cast<uint64_t>(cache->n_kv_heads) * d)
        return fail(GOFANN_ERR_INVALID, "kv_append: a row stride is shorter than its row");
    auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    if ((bits(cache->pages) & 15) || (bits(cache->bounds) & 15))
        return fail(GOFANN_ERR_INVALID, "kv_append: pages and bounds must be 16-byte aligned");
    if ((bits(p.q_out) | bits(p.k_out) | bits(p.v_out)) & 15)
        return fail(GOFANN_ERR_INVALID, "kv_append: outputs must be 16-byte aligned");
    if ((bits(p.q) | bits(p.k) | bits(p.v)) & 1)
        return fail(GOFANN_ERR_INVALID, "kv_append: inputs must be 2-byte aligned");
    if (p.q && p.q == p.q_out && p.q_stride != static_cast<uint64_t>(p.n_heads) * d)
        return fail(GOFANN_ERR_INVALID, "kv_append: q_out may be q only where q's rows are contiguous");
    if (batch->max_pages == 0) return fail(GOFANN_ERR_INVALID, "kv_append: rows without pages");
    // a sequence of n rows touches at most n / 64 + 2 pages, and at most n
    const uint64_t bound = static_cast<uint64_t>(batch->n_rows) / GOFANN_KV_PAGE + 2ull * batch->n_seqs;
    const uint32_t units = static_cast<uint32_t>(bound < batch->n_rows ? bound : batch->n_rows);
    const bool q_wide = (bits(p.q) & 15) == 0 && (p.q_stride & 7) == 0;
    const bool kv_wide = ((bits(p.k) | bits(p.v)) & 15) == 0 && ((p.k_stride | p.v_stride) & 7) == 0;
    // whole lanes of eight dimensions and 16-byte table rows, or the general form
    const bool tables_wide = ((bits(p.cos) | bits(p.sin)) & 15) == 0;
    const int mode = p.rotary_dim == 0 ? kRotateNone
                     : p.rotary_dim % (p.interleaved ? 8 : 16) || !tables_wide ? kRotateAny
                     : p.interleaved                                           ? kRotatePairs
                                                                               : kRotateHalf;
    const dim3 grid(units, cache->n_kv_heads);
    if (d == 64)
        launch_append<64>(*cache, *batch, p, mode, q_wide, kv_wide, grid, as_stream(stream));
    else
        launch_append<128>(*cache, *batch, p, mode, q_wide, kv_wide, grid, as_stream(stream));
    GOFANN_CHECK_LAUNCH("kv_append_kernel");
    return GOFANN_OK;
}

}  // extern "C"
