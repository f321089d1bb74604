// kv_common.cuh — what the cache operators (kv_append.cu, kv_select.cu,
// kv_attention.cu) share: the chunk layout of a 4-bit page, the sequences of
// a call, and the checks of both.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gofann {

constexpr int kKvPage = static_cast<int>(GOFANN_KV_PAGE);
constexpr int kKvGroup = static_cast<int>(GOFANN_KV_GROUP);
constexpr float kNegInf = -__builtin_huge_valf();

// Byte offsets inside the chunk of one (page, head); gofann.h gives the order.
template <int D>
struct KvChunk {
    static constexpr int kGroups = D / kKvGroup;
    static constexpr int kCodes = kKvPage * D / 2;
    static constexpr int kParams = kKvPage * kGroups * 4;
    static constexpr int kKeyParams = kCodes;
    static constexpr int kValueCodes = kCodes + kParams;
    static constexpr int kValueParams = 2 * kCodes + kParams;
    static constexpr int kBytes = 2 * (kCodes + kParams);
};

// Word index of a token's params of group 0 (words of one f16 pair).
template <int D>
__device__ __forceinline__ int kv_param_word(int token)
{
    const int g1 = token >> 4, kt = (token >> 2) & 3, r = (token >> 1) & 1, g0 = token & 1;
    return (((g1 * 2 + g0) * 4 + kt) * 2 + r) * KvChunk<D>::kGroups;
}

// ------------------------------------------------------------- the sequences
// Lengths and rows of a sequence.  A length that the table does not hold
// counts as 0 and offsets that are out of range as no rows: cut to what is in
// range they would move the rows to other positions, where append would write
// over cached tokens.
__device__ __forceinline__ int kv_len(const gofann_kv_batch& b, uint32_t s)
{
    const uint32_t n = __ldg(b.seq_len + s);
    return n <= b.max_pages * GOFANN_KV_PAGE ? static_cast<int>(n) : 0;
}
__device__ __forceinline__ void kv_rows(const gofann_kv_batch& b, uint32_t s, int& first, int& count)
{
    const uint32_t lo = __ldg(b.row_offset + s), hi = __ldg(b.row_offset + s + 1);
    first = static_cast<int>(lo);
    count = lo <= hi && hi <= b.n_rows ? static_cast<int>(hi - lo) : 0;
}

__device__ __forceinline__ void kv_invalid(const gofann_kv_batch& b)
{
    if (b.status) atomicExch(b.status, GOFANN_ERR_INVALID);
}
// Reports such lengths and offsets, the sequences from `s` on in steps.
__device__ __forceinline__ void kv_check_sequences(const gofann_kv_batch& b, uint32_t s, uint32_t step)
{
    for (; s < b.n_seqs; s += step) {
        const uint32_t lo = __ldg(b.row_offset + s), hi = __ldg(b.row_offset + s + 1);
        if (lo > hi || hi > b.n_rows || __ldg(b.seq_len + s) > b.max_pages * GOFANN_KV_PAGE) kv_invalid(b);
    }
}

// The sequence that holds item `flat` when sequence s has count(s) items, and
// the item's place in it.  Every lane of a warp calls it with the same
// `flat`; sequences are taken 32 at a time (one lane each, a warp scan).
// False where the items end before `flat`.
template <class N, class F>
__device__ __forceinline__ bool kv_find(uint32_t n_seqs, N flat, F count, uint32_t& seq, N& at)
{
    const int lane = threadIdx.x & 31;
    for (uint32_t s0 = 0; s0 < n_seqs; s0 += 32) {
        const uint32_t s = s0 + lane;
        const N c = s < n_seqs ? count(s) : N(0);
        N sum = c;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const N v = __shfl_up_sync(kFull, sum, off);
            if (lane >= off) sum += v;
        }
        const unsigned past = __ballot_sync(kFull, flat < sum);
        if (past) {
            const int l = __ffs(past) - 1;
            seq = s0 + l;
            at = flat - __shfl_sync(kFull, sum - c, l);
            return true;
        }
        flat -= __shfl_sync(kFull, sum, 31);
    }
    return false;
}
// Sum of count(s) over the sequences, in every lane of the warp.
template <class N, class F>
__device__ __forceinline__ N kv_total(uint32_t n_seqs, F count)
{
    N sum = 0;
    for (uint32_t s = threadIdx.x & 31; s < n_seqs; s += 32) sum += count(s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
    return sum;
}

// ------------------------------------------------------------------- values
__device__ __forceinline__ float kv_load(const void* p, uint64_t i, int dtype)
{
    if (dtype == GOFANN_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
// Four consecutive elements; `wide`: the address is a multiple of 8 bytes.
__device__ __forceinline__ void kv_load4(const void* p, uint64_t i, int dtype, bool wide, float (&x)[4])
{
    if (wide) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        if (dtype == GOFANN_DTYPE_BF16) {
            x[0] = __uint_as_float(w.x << 16);
            x[1] = __uint_as_float(w.x & 0xffff0000u);
            x[2] = __uint_as_float(w.y << 16);
            x[3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = kv_load(p, i + k, dtype);
    }
}
__device__ __forceinline__ uint32_t kv_pack2(float a, float b, int dtype)
{
    if (dtype == GOFANN_DTYPE_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight consecutive elements as they lie; `wide`: the address is a multiple
// of 16 bytes.
__device__ __forceinline__ uint4 load8(const void* p, uint64_t i, bool wide)
{
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    if (wide) return *reinterpret_cast<const uint4*>(q);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = q[2 * k] | (static_cast<uint32_t>(q[2 * k + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool kBf16>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8])
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (kBf16) {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}
// ----------------------------------------------------------------- the checks
int kv_check(const char* who, const gofann_kv_cache* cache, const gofann_kv_batch* batch, int dtype, uint32_t n_heads);

}  // namespace gofann
