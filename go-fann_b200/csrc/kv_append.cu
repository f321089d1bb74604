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

constexpr int kAppendThreads = 256;

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

// Rotates the vector in `x` (shared, one warp or half warp of lanes per
// vector) and returns the lane's four dimensions d0 .. d0 + 3.
template <int D>
__device__ __forceinline__ void rotate4(const float* x, int d0, const float* cos, const float* sin, int rotary,
                                        bool interleaved, float (&y)[4])
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int d = d0 + k;
        float v = x[d];
        if (d < rotary) {
            const int half = rotary >> 1;
            const int i = interleaved ? d >> 1 : (d < half ? d : d - half);
            const bool low = interleaved ? (d & 1) == 0 : d < half;
            const int other = interleaved ? d ^ 1 : (low ? d + half : d - half);
            const float c = __ldg(cos + i), s = __ldg(sin + i), o = x[other];
            v = low ? __fsub_rn(__fmul_rn(v, c), __fmul_rn(o, s)) : __fadd_rn(__fmul_rn(v, c), __fmul_rn(o, s));
        }
        y[k] = v;
    }
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                   gofann_kv_append_params p, bool q_wide,
                                                                   bool kv_wide)
{
    using Chunk = KvChunk<D>;
    constexpr int G = Chunk::kGroups;
    constexpr int kLanes = D / 4;                       // lanes of one vector
    constexpr int kVectors = kAppendThreads / kLanes;   // vectors at a time
    __shared__ uint8_t codes[2][kKvPage][D];            // keys, values
    __shared__ uint32_t params[2][kKvPage][G];
    __shared__ __align__(16) float stage[kVectors][D];
    __shared__ float top[kAppendThreads / 32];

    const uint32_t head = blockIdx.y;
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && head == 0 && batch.status) {
        for (uint32_t s = threadIdx.x; s < batch.n_seqs; s += kAppendThreads) {
            int first, n;
            kv_rows(batch, s, first, n);
            if (__ldg(batch.seq_len + s) > batch.max_pages * GOFANN_KV_PAGE || n > kv_len(batch, s)) kv_invalid(batch);
        }
    }
    uint32_t seq, at;
    if (!kv_find(batch.n_seqs, blockIdx.x, [&](uint32_t s) { return touched_pages(batch, s); }, seq, at)) return;
    int first_row, n_rows;
    kv_rows(batch, seq, first_row, n_rows);
    const int len = kv_len(batch, seq);
    const int start = len - n_rows;  // position of the first row; negative where rows exceed the length
    const int block = (start > 0 ? start / kKvPage : 0) + static_cast<int>(at);
    const int base = block * kKvPage;
    const int lo = start > base ? start - base : 0;           // first new token of the page
    const int hi = len - base < kKvPage ? len - base : kKvPage;  // tokens that the page holds
    const int32_t page = __ldg(batch.page_table + static_cast<size_t>(seq) * batch.max_pages + block);
    const bool page_ok = page >= 0 && static_cast<uint32_t>(page) < cache.n_pages;
    if (!page_ok && threadIdx.x == 0) kv_invalid(batch);
    uint8_t* chunk = cache.pages + (static_cast<size_t>(page_ok ? page : 0) * cache.n_kv_heads + head) * Chunk::kBytes;

    // ---- rotate and quantise, one vector per kLanes lanes
    const uint32_t group = p.n_heads / cache.n_kv_heads;
    const int n_q = p.q ? static_cast<int>(group) : 0;
    const int per_token = n_q + 2;
    const int work = (hi - lo) * per_token;
    const int vec = threadIdx.x / kLanes, d0 = (threadIdx.x % kLanes) * 4;
    for (int w0 = 0; w0 < work; w0 += kVectors) {
        const int w = w0 + vec;
        const bool on = w < work;
        const int token = on ? lo + w / per_token : lo, kind = on ? w % per_token : 0;
        const int row = first_row + base + token - start;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const bool is_q = kind < n_q, is_k = kind == n_q;
        if (on) {
            if (is_q)
                kv_load4(p.q, static_cast<uint64_t>(row) * p.q_stride + (head * group + kind) * D + d0, p.dtype, q_wide, x);
            else if (is_k)
                kv_load4(p.k, static_cast<uint64_t>(row) * p.k_stride + head * D + d0, p.dtype, kv_wide, x);
            else
                kv_load4(p.v, static_cast<uint64_t>(row) * p.v_stride + head * D + d0, p.dtype, kv_wide, x);
        }
        __syncwarp();
        *reinterpret_cast<float4*>(&stage[vec][d0]) = make_float4(x[0], x[1], x[2], x[3]);
        __syncwarp();
        if (on && (is_q || is_k) && p.rotary_dim) {
            int pos = p.positions ? __ldg(p.positions + row) : base + token;
            if (pos < 0 || static_cast<uint32_t>(pos) >= p.n_positions) {
                if (d0 == 0) kv_invalid(batch);
                pos = 0;
            }
            const size_t t = static_cast<size_t>(pos) * (p.rotary_dim >> 1);
            rotate4<D>(stage[vec], d0, p.cos + t, p.sin + t, static_cast<int>(p.rotary_dim), p.interleaved != 0, x);
        }
        if (on && is_q) {
            uint2* out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.q_out) +
                                                  (static_cast<uint64_t>(row) * p.n_heads + head * group + kind) * D + d0);
            *out = make_uint2(kv_pack2(x[0], x[1], p.dtype), kv_pack2(x[2], x[3], p.dtype));
        }
        // min and max over the 16 lanes of a group (every lane takes part)
        float mn = 0.0f, mx = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = x[k] == x[k] ? fminf(fmaxf(x[k], -GOFANN_KV_CLAMP), GOFANN_KV_CLAMP) : 0.0f;
            mn = k ? fminf(mn, x[k]) : x[k];
            mx = k ? fmaxf(mx, x[k]) : x[k];
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            mn = fminf(mn, __shfl_xor_sync(kFull, mn, off));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, off));
        }
        if (on && !is_q) {
            const __half hs = __float2half_rn(__fdiv_rn(__fsub_rn(mx, mn), 15.0f)), hm = __float2half_rn(mn);
            const float s = __half2float(hs), m = __half2float(hm);
            uint32_t c4 = 0;
            float val[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float c = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[k], m), s)), 0.0f), 15.0f) : 0.0f;
                c4 |= static_cast<uint32_t>(c) << (8 * k);
                val[k] = __fadd_rn(__fmul_rn(c, s), m);
            }
            const int which = is_k ? 0 : 1;
            *reinterpret_cast<uint32_t*>(&codes[which][token][d0]) = c4;
            if ((d0 & (kKvGroup - 1)) == 0) {
                params[which][token][d0 / kKvGroup] = static_cast<uint32_t>(__half_as_ushort(hs)) |
                                                     (static_cast<uint32_t>(__half_as_ushort(hm)) << 16);
            }
            void* out = is_k ? p.k_out : p.v_out;
            if (out)
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) +
                                          (static_cast<uint64_t>(row) * cache.n_kv_heads + head) * D + d0) =
                    make_uint2(kv_pack2(val[0], val[1], p.dtype), kv_pack2(val[2], val[3], p.dtype));
        }
    }
    if (!page_ok) return;
    __syncthreads();

    // ---- merge the codes into the page's words
    uint32_t* kw = reinterpret_cast<uint32_t*>(chunk);
    uint32_t* vw = reinterpret_cast<uint32_t*>(chunk + Chunk::kValueCodes);
    for (int i = threadIdx.x; i < Chunk::kCodes / 4; i += kAppendThreads) {
        // key word [kt][grp][g][t][j]: tokens k0 (even bytes) and k0 + 2, dimensions d .. d + 3
        const int j = i & 3, t = (i >> 2) & 3, g = (i >> 4) & 7, grp = (i >> 7) % G, kt = (i >> 7) / G;
        const int k0 = 16 * (g >> 1) + 4 * kt + (g & 1), d = 64 * grp + 16 * t + 4 * j;
        uint32_t mask = 0, word = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int token = k0 + 2 * r;
            if (token >= lo && token < hi) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(&codes[0][token][d]);
                mask |= 0x00ff00ffu << (8 * r);
                word |= ((c & 0xf) | ((c >> 12) & 0xf0) | ((c << 8) & 0x000f0000) | ((c >> 4) & 0x00f00000)) << (8 * r);
            }
        }
        if (mask) kw[i] = mask == 0xffffffffu ? word : ((kw[i] & ~mask) | word);
        // value word [dt][g][t][kt]: dimensions dv and dv + 8, tokens k1 .. k1 + 3
        const int vkt = i & 3, vt = (i >> 2) & 3, vg = (i >> 4) & 7, dt = i >> 7;
        const int k1 = 16 * vt + 4 * vkt, dv = 16 * dt + vg;
        mask = 0, word = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // token k1 + q = 2 n + e: nibble n of the bytes 2 e + r
            const int token = k1 + q;
            if (token >= lo && token < hi) {
                const int shift = 16 * (q & 1) + 4 * (q >> 1);
                mask |= 0x0f0fu << shift;
                word |= (static_cast<uint32_t>(codes[1][token][dv]) |
                         (static_cast<uint32_t>(codes[1][token][dv + 8]) << 8)) << shift;
            }
        }
        if (mask) vw[i] = mask == 0xffffffffu ? word : ((vw[i] & ~mask) | word);
    }
    uint32_t* kp = reinterpret_cast<uint32_t*>(chunk + Chunk::kKeyParams);
    uint32_t* vp = reinterpret_cast<uint32_t*>(chunk + Chunk::kValueParams);
    for (int i = threadIdx.x; i < kKvPage * G; i += kAppendThreads) {
        const int token = i / G, grp = i % G, w = kv_param_word<D>(token) + grp;
        if (token >= lo && token < hi) {
            kp[w] = params[0][token][grp];
            vp[w] = params[1][token][grp];
        } else if (token < lo) {
            params[0][token][grp] = kp[w];
        }
    }
    // the codes of the keys that the page held before
    if (lo > 0) {
        for (int i = threadIdx.x; i < Chunk::kCodes / 4; i += kAppendThreads) {
            const int j = i & 3, t = (i >> 2) & 3, g = (i >> 4) & 7, grp = (i >> 7) % G, kt = (i >> 7) / G;
            const int k0 = 16 * (g >> 1) + 4 * kt + (g & 1), d = 64 * grp + 16 * t + 4 * j;
            if (k0 >= lo) continue;
            const uint32_t word = kw[i];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (k0 + 2 * r < lo) {
                    const uint32_t b = word >> (8 * r);
                    *reinterpret_cast<uint32_t*>(&codes[0][k0 + 2 * r][d]) =
                        (b & 0xf) | ((b >> 8) & 0xf00) | ((b << 12) & 0xf0000) | ((b << 4) & 0xf000000);
                }
            }
        }
    }
    __syncthreads();

    // ---- bounds of the page's tokens: kThreadsPerDim threads share a dimension
    if (!cache.bounds) return;
    constexpr int kShare = kAppendThreads / D;
    const int d = threadIdx.x / kShare, part = threadIdx.x % kShare;
    float high = kNegInf, low = -kNegInf;
    for (int token = part; token < hi; token += kShare) {
        const uint32_t sm = params[0][token][d / kKvGroup];
        const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffff)));
        const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
        const float x = __fadd_rn(__fmul_rn(static_cast<float>(codes[0][token][d]), s), m);
        high = fmaxf(high, x);
        low = fminf(low, x);
    }
#pragma unroll
    for (int off = 1; off < kShare; off <<= 1) {
        high = fmaxf(high, __shfl_xor_sync(kFull, high, off));
        low = fminf(low, __shfl_xor_sync(kFull, low, off));
    }
    float a = fmaxf(fabsf(high), fabsf(low));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(kFull, a, off));
    if (lane == 0) top[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) a = fmaxf(a, top[w]);
    const float scale = __fdiv_rn(a, 127.0f);
    const size_t entry = static_cast<size_t>(page) * cache.n_kv_heads + head;
    if (part == 0) {
        float h8 = 0.0f, l8 = 0.0f;
        if (scale > 0.0f) {
            h8 = fminf(fmaxf(ceilf(__fdiv_rn(high, scale)), -127.0f), 127.0f);
            l8 = fminf(fmaxf(floorf(__fdiv_rn(low, scale)), -127.0f), 127.0f);
        }
        int8_t* bounds = cache.bounds + entry * 2 * D;
        bounds[d] = static_cast<int8_t>(h8);
        bounds[D + d] = static_cast<int8_t>(l8);
    }
    if (threadIdx.x == 0) cache.bound_scale[entry] = scale;
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
    if ((bits(p.q_out) | bits(p.k_out) | bits(p.v_out)) & 7)
        return fail(GOFANN_ERR_INVALID, "kv_append: outputs must be 8-byte aligned");
    if ((bits(p.q) | bits(p.k) | bits(p.v)) & 1)
        return fail(GOFANN_ERR_INVALID, "kv_append: inputs must be 2-byte aligned");
    if (p.q && p.q == p.q_out && p.q_stride != static_cast<uint64_t>(p.n_heads) * d)
        return fail(GOFANN_ERR_INVALID, "kv_append: q_out may be q only where q's rows are contiguous");
    if (batch->max_pages == 0) return fail(GOFANN_ERR_INVALID, "kv_append: rows without pages");
    // a sequence of n rows touches at most n / 64 + 2 pages, and at most n
    const uint64_t bound = static_cast<uint64_t>(batch->n_rows) / GOFANN_KV_PAGE + 2ull * batch->n_seqs;
    const uint32_t units = static_cast<uint32_t>(bound < batch->n_rows ? bound : batch->n_rows);
    const bool q_wide = (bits(p.q) & 7) == 0 && (p.q_stride & 3) == 0;
    const bool kv_wide = ((bits(p.k) | bits(p.v)) & 7) == 0 && ((p.k_stride | p.v_stride) & 3) == 0;
    const dim3 grid(units, cache->n_kv_heads);
    if (d == 64)
        kv_append_kernel<64><<<grid, kAppendThreads, 0, as_stream(stream)>>>(*cache, *batch, p, q_wide, kv_wide);
    else
        kv_append_kernel<128><<<grid, kAppendThreads, 0, as_stream(stream)>>>(*cache, *batch, p, q_wide, kv_wide);
    GOFANN_CHECK_LAUNCH("kv_append_kernel");
    return GOFANN_OK;
}

}  // extern "C"
