// kv_attention.cuh — what the two attention kernels of the cache share: the
// one for few query columns (kv_attention.cu) and the one for many
// (kv_attention_rows.cu).
#pragma once

#include "kv_async.cuh"

namespace gofann {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x by the special function unit (2 ulp; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Cache blocks that the columns [col0, col0 + cols) of a sequence see.
__device__ __forceinline__ void dense_blocks(const gofann_kv_attention_params& p, int group, int len, int n_rows,
                                             int col0, int cols, int& lo, int& hi)
{
    const int pos0 = len - n_rows + col0 / group, pos1 = len - n_rows + (col0 + cols - 1) / group;
    const int end = p.causal ? pos1 + 1 : len;
    hi = end > 0 && pos1 >= 0 ? (end + kKvPage - 1) / kKvPage : 0;
    const long long low = p.window ? static_cast<long long>(pos0) - p.window + 1 : 0;
    lo = low > 0 ? static_cast<int>(low / kKvPage) : 0;
    if (lo > hi) lo = hi;
}

// The power of two that brings a query column with largest magnitude `top`
// to [2^13, 2^14), as its exponent (from 2^-99 on; smaller ones stay below):
// every f16 within 2^27 of the largest, every bf16 within 2^30, is then an
// exact f16.  The few-column kernel scales half of the elements by another
// 2^-4, which leaves 2^23 and 2^26.
__device__ __forceinline__ int query_exponent(float top)
{
    const int ex = static_cast<int>(__float_as_uint(top) >> 23);
    return 140 - (ex < 28 ? 28 : ex);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// Keys that a row at `pos` sees: low < key <= limit.
__device__ __forceinline__ void row_limits(const gofann_kv_attention_params& p, int pos, int len, int& low, int& limit)
{
    limit = pos < 0 ? -1 : p.causal ? pos : len - 1;
    const long long l = p.window ? static_cast<long long>(pos) - p.window : -1;
    low = l > -1 ? static_cast<int>(l) : -1;
}

// Bits of the tokens of a block that the call shows (key_bits and length).
__device__ __forceinline__ uint64_t shown_tokens(const gofann_kv_attention_params& p, uint32_t seq, int len, int block)
{
    uint64_t shown = ~0ull;
    if (p.key_bits) {
        const uint32_t* bits = p.key_bits + static_cast<size_t>(seq) * p.key_words;
        const uint32_t w = 2u * block;
        shown = (w < p.key_words ? __ldg(bits + w) : 0u) |
                (static_cast<uint64_t>(w + 1 < p.key_words ? __ldg(bits + w + 1) : 0u) << 32);
    }
    const int left = len - block * kKvPage;
    if (left < kKvPage) shown &= left > 0 ? (1ull << left) - 1 : 0ull;
    return shown;
}

// Attention of many query columns per key/value head on the tensor memory
// path (kv_attention_rows.cu).
int attend_rows(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                float* parts, cudaStream_t s);
size_t attend_rows_scratch(uint32_t head_dim, int sms);

}  // namespace gofann
