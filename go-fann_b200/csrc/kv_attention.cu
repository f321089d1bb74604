// kv_attention.cu — attention over the 4-bit cache.
//
// With codes c, scales s and minima m (per token and 64 dimensions),
//   q.k   = sum_grp s_grp (q_grp . c_grp) + m_grp (sum of q_grp)
//   sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)
// so the matrix instructions read the codes themselves.  A code word masked
// to nibbles is already a pair of f16 numbers: 0x000c is the subnormal
// c * 2^-24 and 0x00c0 is c * 2^-20, both exact, so four ANDs and a shift turn
// a word of eight codes into the lane's A operand of a 16 x 8 x 16 product.
// The 2^-24 goes into an f32 scale, the extra 2^4 of the odd nibbles into the
// other operand.
//
// Tokens are the rows (M = 16) and query heads the columns (N = 8) of both
// products: S^T = K Q^T, then O^T = V^T P^T; the transposition of P between
// the two layouts is one movmatrix per 8 x 8 tile.
#include "kv_attention.cuh"

namespace gofann {
namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float* c)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// (a, b) += c, two f32 sums in one instruction.
__device__ __forceinline__ void add_pair(float& a, float& b, const float* c)
{
    asm("{\n\t.reg .b64 x, y;\n\t"
        "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(c[0]), "f"(c[1]));
}
// The A operand of 16 rows x 16 steps from one word of eight codes.
__device__ __forceinline__ void code_operand(uint32_t w, uint32_t (&a)[4])
{
    a[0] = w & 0x000f000fu;
    a[2] = w & 0x00f000f0u;
    w >>= 8;
    a[1] = w & 0x000f000fu;
    a[3] = w & 0x00f000f0u;
}
__device__ __forceinline__ float2 both_halves(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// N (1, 2 or 4) words from an address that is a multiple of 4 N.
template <int N>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[N])
{
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A call's parameters, and the units that every tile counts where that is the
// same number for all of them (0 = each sequence has its own).
struct Call : gofann_kv_attention_params {
    int fixed;
};

// The query columns that a warp works on at a time: rows of a sequence x
// query heads of one key/value head.
struct Tile {
    uint32_t seq;
    int first_row, n_rows, len;  // of the sequence
    int col0, cols;              // columns of the sequence (dense) or of the row (selected)
    int row;                     // selected: the row inside the sequence
};

// A sequence's share of the work in units of one cache block for one tile and
// key/value head: every tile counts `span` blocks from `lo` on (what all of
// the sequence's rows see), at least one, so that each tile has an owner.
struct SeqWork {
    int tiles, lo, span;
};
template <bool kSelected>
__device__ __forceinline__ SeqWork seq_work(const gofann_kv_batch& b, const Call& p, int group,
                                            int width, uint32_t s)
{
    int first, n, lo = 0, hi = static_cast<int>(p.n_select);
    kv_rows(b, s, first, n);
    SeqWork w{0, 0, 1};
    if (n == 0) return w;
    if (kSelected) {
        w.tiles = n * ((group + width - 1) / width);
    } else {
        w.tiles = (n * group + width - 1) / width;
        dense_blocks(p, group, kv_len(b, s), n, 0, n * group, lo, hi);
    }
    w.lo = lo;
    w.span = p.fixed ? p.fixed : hi > lo ? hi - lo : 1;
    return w;
}

// A (tile, head) and its place among all units.
struct Item {
    Tile tile;
    uint32_t head;
    uint64_t begin, end;
};

// The sequence that the units around a point belong to.
struct SeqCursor {
    uint32_t seq;
    uint64_t begin, end;
    int lo, span;
};

template <bool kSelected>
__device__ __forceinline__ void make_tile(const gofann_kv_batch& b, const Call& p, int group,
                                          int width, uint32_t seq, int at, Tile& tile)
{
    tile.seq = seq;
    kv_rows(b, seq, tile.first_row, tile.n_rows);
    tile.len = kv_len(b, seq);
    if (kSelected) {
        const int per_row = (group + width - 1) / width;
        tile.row = at / per_row;
        tile.col0 = at % per_row * width;
        tile.cols = group - tile.col0 < width ? group - tile.col0 : width;
    } else {
        const int total = tile.n_rows * group;
        tile.row = 0;
        tile.col0 = at * width;
        tile.cols = total - tile.col0 < width ? total - tile.col0 : width;
    }
}

template <bool kSelected>
__device__ __forceinline__ uint64_t total_units(const gofann_kv_batch& b, const Call& p,
                                                uint32_t n_kv, int group, int width)
{
    return kv_total<uint64_t>(b.n_seqs, [&](uint32_t s) {
        const SeqWork w = seq_work<kSelected>(b, p, group, width, s);
        return static_cast<uint64_t>(w.tiles) * n_kv * w.span;
    });
}
// The sequence of unit `flat`; false past the end.
template <bool kSelected>
__device__ __forceinline__ bool seek(const gofann_kv_batch& b, const Call& p, uint32_t n_kv,
                                     int group, int width, uint64_t flat, SeqCursor& c)
{
    uint64_t at;
    const auto units = [&](uint32_t s) {
        const SeqWork w = seq_work<kSelected>(b, p, group, width, s);
        return static_cast<uint64_t>(w.tiles) * n_kv * w.span;
    };
    if (!kv_find<uint64_t>(b.n_seqs, flat, units, c.seq, at)) return false;
    const SeqWork w = seq_work<kSelected>(b, p, group, width, c.seq);
    c.begin = flat - at;
    c.end = c.begin + static_cast<uint64_t>(w.tiles) * n_kv * w.span;
    c.lo = w.lo;
    c.span = w.span;
    return true;
}
// The sequence of the unit that `place` names once it knows the number of all
// units; false where it names one past the end.
template <bool kSelected, class F>
__device__ __forceinline__ bool seek_by_total(const gofann_kv_batch& b, const Call& p, uint32_t n_kv, int group, int width,
                                              F place, SeqCursor& c)
{
    if (b.n_seqs > 32) {
        const uint64_t flat = place(total_units<kSelected>(b, p, n_kv, group, width));
        return seek<kSelected>(b, p, n_kv, group, width, flat, c);
    }
    // one look at the sequences is enough
    const int lane = threadIdx.x & 31;
    SeqWork w{0, 0, 1};
    if (lane < static_cast<int>(b.n_seqs)) w = seq_work<kSelected>(b, p, group, width, lane);
    const uint64_t units = static_cast<uint64_t>(w.tiles) * n_kv * w.span;
    uint64_t upto = units;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint64_t v = __shfl_up_sync(kFull, upto, off);
        if (lane >= off) upto += v;
    }
    const uint64_t flat = place(__shfl_sync(kFull, upto, 31));
    const unsigned past = __ballot_sync(kFull, flat < upto);
    if (!past) return false;
    const int l = __ffs(past) - 1;
    c.seq = l;
    c.end = __shfl_sync(kFull, upto, l);
    c.begin = c.end - __shfl_sync(kFull, units, l);
    c.lo = __shfl_sync(kFull, w.lo, l);
    c.span = __shfl_sync(kFull, w.span, l);
    return true;
}
// The next sequence that has units (the caller knows that there is one).
template <bool kSelected>
__device__ __forceinline__ void next_sequence(const gofann_kv_batch& b, const Call& p,
                                              uint32_t n_kv, int group, int width, SeqCursor& c)
{
    while (c.seq + 1 < b.n_seqs) {
        const SeqWork w = seq_work<kSelected>(b, p, group, width, ++c.seq);
        if (w.tiles == 0) continue;
        c.begin = c.end;
        c.end = c.begin + static_cast<uint64_t>(w.tiles) * n_kv * w.span;
        c.lo = w.lo;
        c.span = w.span;
        return;
    }
}
// a / b: 64-bit numbers take a routine, most are short.
__device__ __forceinline__ uint64_t divide(uint64_t a, uint32_t b)
{
    return a >> 32 ? a / b : static_cast<uint32_t>(a) / b;
}

template <bool kSelected>
__device__ __forceinline__ void make_item(const gofann_kv_batch& b, const Call& p, uint32_t n_kv,
                                          int group, int width, uint64_t flat, const SeqCursor& c, Item& item)
{
    const uint64_t i = divide(flat - c.begin, c.span), tile = divide(i, n_kv);
    item.begin = c.begin + i * c.span;
    item.end = item.begin + c.span;
    item.head = static_cast<uint32_t>(i - tile * n_kv);
    make_tile<kSelected>(b, p, group, width, c.seq, static_cast<int>(tile), item.tile);
}

// Running softmax state of one warp for columns 2t, 2t + 1 of each 8-column
// tile and dimensions 16 dt + g, + 8.  All sums are in units of the weights
// 2^(logit - base), base = reference - (kUp - e) in log2 units: e is the
// largest exponent of a value scale so far, so the products weight * scale are
// below 2^8 at the reference, below 2^15 where a logit is kLag above it, and
// f16 holds them down to 2^-24 whatever the values' magnitude.
constexpr int kUp = 22;
constexpr float kLag = 7.0f;
template <int D, int NT>
struct State {
    float m[NT][2];                      // reference, in the query column's own unit
    float l[NT][2];                      // this lane's part of the sum of weights
    float z[NT][2][KvChunk<D>::kGroups]; // this lane's part of sum w * (minimum + 8 scale)
    float o[D / 16][NT][4];              // sum (w * scale) * (code - 8) * 2^-24
    int e;
};

template <int D, int NT>
__device__ __forceinline__ void clear(State<D, NT>& st)
{
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            st.m[n][c] = kNegInf;
            st.l[n][c] = 0.0f;
#pragma unroll
            for (int grp = 0; grp < KvChunk<D>::kGroups; ++grp) st.z[n][c][grp] = 0.0f;
        }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) st.o[dt][n][i] = 0.0f;
    st.e = 1;
}

// The query columns as B operands and their f32 companions.  A column's
// logits are `unit` (log2 units) times its product with the key.
template <int D, int NT>
struct Query {
    uint32_t b[D / 16][NT][2];
    float unit[NT][2], lag[NT][2];          // lag: kLag in the column's unit
    float sum[NT][2][KvChunk<D>::kGroups];  // sum of the column over a group
    int limit[NT][2], low[NT][2];           // keys seen: low < key <= limit
};

// Scores of a page's 64 tokens x 8 NT columns from the key half of a chunk.
// This lane's tokens are first + 2 i, i = 0 .. 7.  kMask: 0 = every column
// sees every token, 1 = every column sees the tokens whose bit `shown` has,
// 2 = each column has limits of its own too.
template <int D, int NT, int kMask>
__device__ __forceinline__ void page_scores(const unsigned char* keys, const Query<D, NT>& q, int key0, uint64_t shown,
                                            float (&s)[4][NT][4])
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        uint32_t kp[2 * G];  // tokens first + 4 kt, + 2
        load_words<2 * G>(keys + KvChunk<D>::kKeyParams + (g * 4 + kt) * 8 * G, kp);
        float acc[G][NT][4];
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            const uint4 w4 = reinterpret_cast<const uint4*>(keys)[(kt * G + grp) * 32 + lane];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a[4];
                code_operand(w[j], a);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t(&b)[2] = q.b[grp * 4 + j][n];
                    mma_f16(acc[grp][n], a, b[0], b[1], j == 0 ? zero : acc[grp][n]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float2 sm[G];
#pragma unroll
            for (int grp = 0; grp < G; ++grp) sm[grp] = both_halves(kp[r * G + grp]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = sm[0].y * q.sum[n][c][0];
#pragma unroll
                    for (int grp = 1; grp < G; ++grp) x = fmaf(sm[grp].y, q.sum[n][c][grp], x);
#pragma unroll
                    for (int grp = 0; grp < G; ++grp) x = fmaf(sm[grp].x, acc[grp][n][2 * r + c], x);
                    s[kt][n][2 * r + c] = x;
                }
        }
    }
    if constexpr (kMask > 0) {
        const int first = 16 * (g >> 1) + (g & 1);
        const uint32_t mine = static_cast<uint32_t>(shown >> first);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const bool on = (mine >> (4 * kt + 2 * r)) & 1;
                const int key = key0 + first + 4 * kt + 2 * r;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        if (!on || (kMask == 2 && (key > q.limit[n][c] || key <= q.low[n][c]))) s[kt][n][2 * r + c] = kNegInf;
            }
    }
}

// Softmax update and weighted values from the value half of a chunk.
template <int D, int NT, int kMask>
__device__ __forceinline__ void page_values(const unsigned char* values, const Query<D, NT>& q, uint64_t shown,
                                            float (&s)[4][NT][4], State<D, NT>& st)
{
    constexpr int G = KvChunk<D>::kGroups, kAt = KvChunk<D>::kCodes;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const uint32_t mine = static_cast<uint32_t>(shown >> (16 * (g >> 1) + (g & 1)));

    // ---- the largest value scale; a hidden token's params may be anything,
    // so they count as 0 here and below
    const uint32_t* params = reinterpret_cast<const uint32_t*>(values + kAt) + g * 8 * G;
    __half2 top = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
    for (int i = 0; i < 2 * G; ++i) {
        uint32_t w[4];
        load_words<4>(reinterpret_cast<const unsigned char*>(params + 4 * i), w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (kMask > 0 && !((mine >> (2 * ((4 * i + k) / G))) & 1)) w[k] = 0;
            top = __hmax2(top, *reinterpret_cast<const __half2*>(&w[k]));
        }
    }
    const int e_here = static_cast<int>((*reinterpret_cast<const uint32_t*>(&top) & 0x7c00u) >> 10);

    // ---- the reference of the weights: it moves only where a score is kLag
    // above it, there is none yet, or a value scale has a larger exponent
    float local[NT][2];
    bool far = e_here > st.e;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(s[0][n][c], s[0][n][2 + c]);
#pragma unroll
            for (int kt = 1; kt < 4; ++kt) mx = fmaxf(mx, fmaxf(s[kt][n][c], s[kt][n][2 + c]));
            local[n][c] = mx;
            far |= mx > st.m[n][c] + q.lag[n][c];
        }
    if (__any_sync(kFull, far)) {
        const int e = max(st.e, static_cast<int>(__reduce_max_sync(kFull, static_cast<unsigned>(e_here))));
        const float shift = static_cast<float>(e - st.e);
        st.e = e;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float mx = fmaxf(local[n][c], st.m[n][c]);
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
                const float use = mx == kNegInf ? 0.0f : mx;
                const float f = exp2_fast(fmaf(st.m[n][c] - use, q.unit[n][c], -shift));
                st.m[n][c] = mx;
                st.l[n][c] *= f;
#pragma unroll
                for (int grp = 0; grp < G; ++grp) st.z[n][c][grp] *= f;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) st.o[dt][n][2 * r + c] *= f;
            }
    }
    const float up = static_cast<float>(kUp - st.e);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float unit = q.unit[n][c], base = fmaf(st.m[n][c] == kNegInf ? 0.0f : st.m[n][c], unit, -up);
            float l = st.l[n][c];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x = exp2_fast(fmaf(s[kt][n][2 * r + c], unit, -base));
                    s[kt][n][2 * r + c] = x;
                    l += x;
                }
            st.l[n][c] = l;
        }

    // ---- weighted values.  The matrix instruction truncates its sums, so a
    // long chain of the codes' one-sided products would drift: codes are
    // centred (8 times the sum of the weights is taken off by the same
    // instruction on a constant operand) and a page's sum joins the running
    // one by an f32 addition.
    const uint32_t eight[4] = {0x80088008u, 0x80088008u, 0x80808080u, 0x80808080u};  // -8 * 2^-24, -8 * 2^-20
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
        uint32_t b[4][NT][2];
        float centre[NT][4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                uint32_t w = params[(2 * kt + r) * G + grp];
                if (kMask > 0 && !((mine >> (4 * kt + 2 * r)) & 1)) w = 0;
                const float2 sm = both_halves(w);
                const float vs = r ? sm.x * 0.0625f : sm.x, vm = fmaf(8.0f, sm.x, sm.y);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float p0 = s[kt][n][2 * r], p1 = s[kt][n][2 * r + 1];
                    st.z[n][0][grp] = fmaf(p0, vm, st.z[n][0][grp]);
                    st.z[n][1][grp] = fmaf(p1, vm, st.z[n][1][grp]);
                    b[kt][n][r] = transpose8x8(pack_f16(p0 * vs, p1 * vs));
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(centre[n], eight, b[kt][n][0], b[kt][n][1], kt == 0 ? zero : centre[n]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dt = grp * 4 + i;
            float acc[NT][4];
            const uint4 w4 = reinterpret_cast<const uint4*>(values)[dt * 32 + lane];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t a[4];
                code_operand(w[kt], a);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(acc[n], a, b[kt][n][0], b[kt][n][1], kt == 0 ? centre[n] : acc[n]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; k += 2) add_pair(st.o[dt][n][k], st.o[dt][n][k + 1], acc[n] + k);
        }
    }
}

template <int D, int NT>
__device__ __forceinline__ void load_query(const Call& p, const Tile& tile, uint32_t head,
                                           int group, bool selected, bool wide, Query<D, NT>& q)
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // a negative scale turns the query around, a scale of 0 makes it 0
    const float sign = p.scale < 0.0f ? -1.0f : p.scale > 0.0f ? 1.0f : 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        // this lane's column g: 16 dimensions of each group
        const int c = n * 8 + g;
        float x[G][4][4];
        float top = 0.0f;
        if (c < tile.cols) {
            const int col = tile.col0 + c;
            const int row = tile.first_row + (selected ? tile.row : col / group);
            const uint64_t at = static_cast<uint64_t>(row) * p.q_stride +
                                static_cast<uint64_t>(head * group + (selected ? col : col % group)) * D + 16 * t;
#pragma unroll
            for (int grp = 0; grp < G; ++grp)
#pragma unroll
                for (int j = 0; j < 4; ++j) kv_load4(p.q, at + grp * 64 + 4 * j, p.dtype, wide, x[grp][j]);
        } else {
#pragma unroll
            for (int grp = 0; grp < G; ++grp)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[grp][j][k] = 0.0f;
        }
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) top = fmaxf(top, fabsf(x[grp][j][k]));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
        const int ex = query_exponent(top);
        const float down = power_of_two(ex) * sign;
        float sum[G];
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            sum[grp] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    y[k] = x[grp][j][k] * down;
                    sum[grp] += y[k];
                }
                q.b[grp * 4 + j][n][0] = pack_f16(y[0], y[1]);
                q.b[grp * 4 + j][n][1] = pack_f16(y[2] * 0.0625f, y[3] * 0.0625f);
            }
            sum[grp] += __shfl_xor_sync(kFull, sum[grp], 1);
            sum[grp] += __shfl_xor_sync(kFull, sum[grp], 2);
            sum[grp] *= 0x1p-24f;  // the unit of the codes' products
        }
        // undoes `down` and the codes' subnormals
        const float undo = p.scale == 0.0f ? 1.0f : fmaxf(fabsf(p.scale) * kLog2e * power_of_two(-ex) * 0x1p24f, FLT_MIN);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            q.unit[n][e] = __shfl_sync(kFull, undo, 4 * (2 * t + e));
            q.lag[n][e] = fminf(kLag / q.unit[n][e], FLT_MAX);
#pragma unroll
            for (int grp = 0; grp < G; ++grp) q.sum[n][e][grp] = __shfl_sync(kFull, sum[grp], 4 * (2 * t + e));
            const int cc = n * 8 + 2 * t + e;
            const int row = selected ? tile.row : (tile.col0 + cc) / group;
            row_limits(p, tile.len - tile.n_rows + row, tile.len, q.low[n][e], q.limit[n][e]);
            if (cc >= tile.cols) {  // no mask of its own: nothing of it is written
                q.limit[n][e] = 0x7fffffff;
                q.low[n][e] = -1;
            }
        }
    }
}

// The place of the next half chunk in a ring and the parity of its barrier.
template <int kSlots>
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next()
    {
        if (++slot == kSlots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// What a warp keeps in shared memory to spare registers: the items of its
// partial results (end 0 = none), the one in work, where its loads and its
// work are.
struct WarpItems {
    Item part[2], now;  // part: the first item, the last
    SeqCursor ahead, here;
};

// A thread block's warps and shared memory: per warp a ring of half chunks
// (keys or values), the place of its first partial result (the last one takes
// the ring's), its items.  Two partial results a warp are enough because its
// units are consecutive.
template <int D, int NT>
struct Attend {
    static constexpr int kCols = 8 * NT;
    // 128, 168 or 255 registers a thread.  Instead with 8 warps: 32 rows over
    // 32768 tokens, head_dim 128, 8 columns, 183 us (12 warps: 170); 509 rows of
    // 32 selected blocks, head_dim 64, 107 us (16 warps: 86).
    static constexpr int kWarps = D * NT == 64 ? 16 : D * NT == 128 ? 12 : 8;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kHalf = KvChunk<D>::kBytes / 2;
    static constexpr int kSlots = D == 64 || NT == 2 ? 4 : 3;
    static constexpr int kPart = kCols * (D + 4) + 2 * kCols;  // floats: values, max, sum
    static constexpr size_t kRing = static_cast<size_t>(kWarps) * kSlots * kHalf;
    static constexpr size_t kFirst = sizeof(float) * kWarps * kPart;
    static constexpr size_t kItems = sizeof(WarpItems) * kWarps;
    static constexpr size_t kFactors = sizeof(float) * kCols * 34;
    static constexpr size_t kBytes = kRing + kFirst + kItems + kFactors + sizeof(uint64_t) * kWarps * kSlots;
    static_assert(2 * kWarps <= 32 && sizeof(float) * kPart <= kSlots * kHalf, "a warp's last partial result takes its ring's place");
    static_assert(kBytes <= 227 * 1024, "shared memory of a block");
};

// Units of one block: a share of the total, at least one per warp, and whole
// items where all count the same (then no item has to be joined).
__device__ __forceinline__ uint64_t units_per_block(uint64_t total, uint32_t blocks, int warps, int fixed)
{
    if (fixed) return divide(divide(total, fixed) + blocks - 1, blocks) * fixed;
    const uint64_t c = divide(total + blocks - 1, blocks);
    return c > warps ? c : warps;
}

// A block's partial result in scratch: [cols] max, [cols] sum, [cols][D]
// values; two per block (its first item, and its last if that is another).
template <int D, int NT>
constexpr size_t kPartFloats = 8 * NT * (D + 2);

// A row's sum of weights is 0 where it sees no key, and no number where its
// query holds one that is none, which its output then shows.
template <int D>
__device__ __forceinline__ void store_row(const Call& p, const Tile& tile, uint32_t head, int group,
                                          bool selected, int c, int d, float m, float l, const float (&o)[4])
{
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int col = tile.col0 + c;
    const uint64_t row = tile.first_row + (selected ? tile.row : col / group);
    const uint64_t at = row * p.n_heads + head * group + (selected ? col : col % group);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * D + d) =
        l != 0.0f ? make_uint2(kv_pack2(o[0] * inv, o[1] * inv, p.dtype), kv_pack2(o[2] * inv, o[3] * inv, p.dtype))
                  : make_uint2(0u, 0u);
    if (d == 0 && p.lse) p.lse[at] = l != 0.0f ? (m + log2f(l)) * kLn2 : kNegInf;
}

// The rows of a whole item from the lanes that hold them: pairs of columns
// become pairs of dimensions by the transposition that P takes.
template <int D, int NT, bool kSelected>
__device__ __forceinline__ void store_item(const Call& p, const Tile& tile, uint32_t head, int group,
                                           const State<D, NT>& st)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const auto place = [&](int c) {
        const int col = tile.col0 + c;
        const uint64_t row = tile.first_row + (kSelected ? tile.row : col / group);
        return row * p.n_heads + head * group + (kSelected ? col : col % group);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float inv[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float l = st.l[n][c];
            inv[c] = l != 0.0f ? 1.0f / l : 0.0f;
            if (g == 0 && p.lse && n * 8 + 2 * t + c < tile.cols)
                p.lse[place(n * 8 + 2 * t + c)] = l != 0.0f ? (st.m[n][c] + log2f(l)) * kLn2 : kNegInf;
        }
        const bool on = n * 8 + g < tile.cols;
        uint16_t* out = static_cast<uint16_t*>(p.out) + (on ? place(n * 8 + g) : 0) * D;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float a = inv[0] != 0.0f ? st.o[dt][n][2 * r] * inv[0] : 0.0f;
                const float b = inv[1] != 0.0f ? st.o[dt][n][2 * r + 1] * inv[1] : 0.0f;
                const uint32_t w = transpose8x8(kv_pack2(a, b, p.dtype));
                if (on) *reinterpret_cast<uint32_t*>(out + dt * 16 + 8 * r + 2 * t) = w;
            }
    }
}

// What the 32 units from a multiple of 32 after a warp's first one read: lane
// i has unit i's chunk (or nullptr) and cache block; `valid` has their bits.
struct Batch32 {
    const unsigned char* chunk;
    int block;
    unsigned valid;
};

template <int D, int NT, bool kSelected>
__device__ __forceinline__ void look_up(const gofann_kv_cache& cache, const gofann_kv_batch& b,
                                        const Call& p, int group, uint64_t flat0, uint64_t end,
                                        SeqCursor& c, Batch32& got)
{
    constexpr int kCols = 8 * NT;
    const uint64_t flat = flat0 + (threadIdx.x & 31);
    const uint32_t n_kv = cache.n_kv_heads;
    bool todo = flat < end;
    got.chunk = nullptr;
    got.block = 0;
    while (true) {
        if (todo && flat < c.end) {
            todo = false;
            const uint64_t at = flat - c.begin, i = divide(at, c.span), tile_at = divide(i, n_kv);
            const uint32_t head = static_cast<uint32_t>(i - tile_at * n_kv);
            int block = c.lo + static_cast<int>(at - i * c.span);
            Tile tile;
            make_tile<kSelected>(b, p, group, kCols, c.seq, static_cast<int>(tile_at), tile);
            bool on = true;
            if (kSelected) {
                block = __ldg(p.selected +
                              (static_cast<size_t>(tile.first_row + tile.row) * n_kv + head) * p.n_select + block);
                on = block >= 0 && block < (tile.len + kKvPage - 1) / kKvPage;
            } else {
                int lo, hi;
                dense_blocks(p, group, tile.len, tile.n_rows, tile.col0, tile.cols, lo, hi);
                on = block >= lo && block < hi;
            }
            if (on) {
                const int32_t page = __ldg(b.page_table + static_cast<size_t>(c.seq) * b.max_pages + block);
                if (page < 0 || static_cast<uint32_t>(page) >= cache.n_pages) {
                    kv_invalid(b);
                } else {
                    got.chunk = cache.pages + (static_cast<size_t>(page) * n_kv + head) * KvChunk<D>::kBytes;
                    got.block = block;
                }
            }
        }
        if (!__any_sync(kFull, todo)) break;
        next_sequence<kSelected>(b, p, n_kv, group, kCols, c);
    }
    got.valid = __ballot_sync(kFull, got.chunk != nullptr);
}

// Each thread block takes an equal share of all units, each warp an equal,
// consecutive part of the share; a warp that has a whole item writes its rows
// itself.
//
// What bounds it: the instructions that turn codes into operands and join a
// page's sums (a warp issues 94 M of them for 0.81 GB), whose fixed latencies
// 12 to 16 warps hide in part; 54 % of the issue slots are taken.  32 rows over
// 32768 tokens (64 query, 8 key/value heads of 128) take 186 us, 4.4 TB/s, 0.67
// of the measured copy (170 to 186 from one device to the next); one row over
// 131072 tokens 53 us, of which the
// partial results' join is 8; 48 rows of 64 selected blocks 70 us, 3.2 TB/s:
// each (row, head) has its own list of pages to look up and its own join.
template <int D, int NT, bool kSelected>
__global__ void __launch_bounds__(Attend<D, NT>::kThreads, 1) kv_attend_kernel(gofann_kv_cache cache,
                                                                               gofann_kv_batch batch,
                                                                               Call p, bool wide,
                                                                               float* __restrict__ parts)
{
    using Cfg = Attend<D, NT>;
    constexpr int G = KvChunk<D>::kGroups, kCols = Cfg::kCols, kWarps = Cfg::kWarps, kSlots = Cfg::kSlots;
    constexpr int kHalf = Cfg::kHalf, kPart = Cfg::kPart;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + static_cast<size_t>(warp) * kSlots * kHalf;
    const auto first_part = [&](int w) { return reinterpret_cast<float*>(smem + Cfg::kRing) + w * kPart; };
    const auto last_part = [&](int w) { return reinterpret_cast<float*>(smem + static_cast<size_t>(w) * kSlots * kHalf); };
    WarpItems* warp_items = reinterpret_cast<WarpItems*>(smem + Cfg::kRing + Cfg::kFirst);
    WarpItems& mine = warp_items[warp];
    float* factors = reinterpret_cast<float*>(smem + Cfg::kRing + Cfg::kFirst + Cfg::kItems);  // [cols][32], max, sum
    const uint32_t bars = shared_addr(smem + Cfg::kRing + Cfg::kFirst + Cfg::kItems + Cfg::kFactors) + warp * kSlots * 8;
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const uint32_t n_kv = cache.n_kv_heads;

    if (lane < kSlots) barrier_init(bars + 8 * lane, 1);
    barrier_fence();
    launch_next();
    if (lane < 2) mine.part[lane].end = 0;
    __syncwarp();
    uint64_t u0 = 0, u1 = 0, w0 = 0, w1 = 0;  // units of the block, of the warp
    SeqCursor from;
    seek_by_total<kSelected>(
        batch, p, n_kv, group, kCols,
        [&](uint64_t total) {
            const uint64_t share = units_per_block(total, gridDim.x, kWarps, p.fixed);
            u0 = share * blockIdx.x;
            u1 = u0 + share < total ? u0 + share : total;
            if (u0 >= u1) return ~0ull;
            const uint64_t per_warp = divide(u1 - u0 + kWarps - 1, kWarps);
            w0 = u0 + warp * per_warp;
            w1 = w0 + per_warp < u1 ? w0 + per_warp : u1;
            return static_cast<unsigned long long>(w0 < w1 ? w0 : ~0ull);
        },
        from);
    if (blockIdx.x == 0) kv_check_sequences(batch, threadIdx.x, Cfg::kThreads);
    if (u0 >= u1) return;

    bool alive = true;  // false once a wait has run out
    if (w0 < w1) {
        Batch32 now, then;
        {
            SeqCursor c = from;
            if (lane == 0) mine.here = c;
            // the first item's queries come while the pages are looked up
            Item item;
            make_item<kSelected>(batch, p, n_kv, group, kCols, w0, c, item);
            if (lane < item.tile.cols * 2) {
                const int col = item.tile.col0 + lane / 2;
                const int row = item.tile.first_row + (kSelected ? item.tile.row : col / group);
                prefetch_l1(static_cast<const uint16_t*>(p.q) + static_cast<uint64_t>(row) * p.q_stride +
                            static_cast<uint64_t>(item.head * group + (kSelected ? col : col % group)) * D + (lane & 1) * (D / 2));
            }
            look_up<D, NT, kSelected>(cache, batch, p, group, w0, w1, c, now);
            if (lane == 0) mine.ahead = c;
            __syncwarp();
        }
        then.valid = 0;
        // half chunks in order: the valid units' keys and values.  `todo` has
        // the units of a batch that are still to be loaded; a unit's own lane
        // issues its loads.
        Ring<kSlots> in, out;
        int flight = 0;           // halves issued and not yet taken
        unsigned todo = now.valid, todo_then = 0;
        int values_lane = -1;     // the lane whose chunk's values come next
        const unsigned char* src = nullptr;
        const auto fill = [&]() {  // loads what the free slots hold
            while (flight < kSlots) {
                int l = values_lane;
                int half = kHalf;
                if (l < 0) {
                    if (!(todo | todo_then)) return;
                    const bool in_now = todo != 0;
                    l = __ffs(in_now ? todo : todo_then) - 1;
                    if (in_now) todo &= todo - 1; else todo_then &= todo_then - 1;
                    if (lane == l) src = in_now ? now.chunk : then.chunk;
                    half = 0;
                    values_lane = l;
                } else {
                    values_lane = -1;
                }
                if (lane == l) {
                    barrier_expect(bars + 8 * in.slot, kHalf);
                    bulk_load(shared_addr(ring) + in.slot * kHalf, src + half, kHalf, bars + 8 * in.slot);
                }
                in.next();
                ++flight;
            }
        };
        const auto take = [&]() { return barrier_wait(bars + 8 * out.slot, out.phase); };
        const auto release = [&]() {
            out.next();
            --flight;
            __syncwarp();
        };
        fill();

        uint64_t flat = w0;
        while (flat < w1) {
            // ---- one item, or this warp's part of it
            {
                SeqCursor c = mine.here;
                Item item;
                __syncwarp();
                while (flat >= c.end) next_sequence<kSelected>(batch, p, n_kv, group, kCols, c);
                make_item<kSelected>(batch, p, n_kv, group, kCols, flat, c, item);
                if (lane == 0) {
                    mine.here = c;
                    mine.now = item;
                }
                __syncwarp();
            }
            const Item& item = mine.now;
            const Tile& tile = item.tile;
            const int len = tile.len;
            const uint64_t start = flat, stop = item.end < w1 ? item.end : w1;
            Query<D, NT> q;
            load_query<D, NT>(p, tile, item.head, group, kSelected, wide, q);
            // keys in (low, limit] are seen by every column; `alike`: by the
            // same token, no column sees another key
            int limit = 0x7fffffff, low = -1, limit_most = -1, low_least = 0x7fffffff;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    limit = min(limit, q.limit[n][e]);
                    low = max(low, q.low[n][e]);
                    if (n * 8 + 2 * t + e < tile.cols) {
                        limit_most = max(limit_most, q.limit[n][e]);
                        low_least = min(low_least, q.low[n][e]);
                    }
                }
            limit = __reduce_min_sync(kFull, limit);
            low = __reduce_max_sync(kFull, low);
            const bool alike = limit == __reduce_max_sync(kFull, limit_most) && low == __reduce_min_sync(kFull, low_least);
            State<D, NT> st;
            clear(st);
            const uint32_t seq = tile.seq;
#pragma unroll 1
            for (; flat < stop; ++flat) {
                const int l = static_cast<int>(flat - w0) & 31;
                if (l == 0) {
                    // the next 32 units are looked up a batch ahead of their loads
                    if (flat != w0) {
                        now = then;
                        todo = todo_then;
                    }
                    then.valid = 0;
                    if (flat + 32 < w1) {
                        SeqCursor c = mine.ahead;
                        __syncwarp();
                        look_up<D, NT, kSelected>(cache, batch, p, group, flat + 32, w1, c, then);
                        if (lane == 0) mine.ahead = c;
                        __syncwarp();
                    }
                    todo_then = then.valid;
                    fill();  // there may have been nothing to load until here
                }
                if (!((now.valid >> l) & 1) || !alive) continue;
                const int block = __shfl_sync(kFull, now.block, l), key0 = block * kKvPage;
                uint64_t shown = shown_tokens(p, seq, len, block);
                const bool edge = key0 + kKvPage - 1 > limit || key0 <= low;
                if (edge && alike) {
                    const int a = limit - key0, b = low - key0;
                    shown &= a < 0 ? 0ull : a >= 63 ? ~0ull : (2ull << a) - 1;
                    shown &= b < 0 ? ~0ull : b >= 63 ? 0ull : ~((2ull << b) - 1);
                }
                const int mask = edge && !alike ? 2 : shown != ~0ull ? 1 : 0;
                float s[4][NT][4];
                alive = take();
                if (!alive) continue;
                if (shown != 0) {
                    if (mask == 0)
                        page_scores<D, NT, 0>(ring + out.slot * kHalf, q, key0, shown, s);
                    else if (mask == 1)
                        page_scores<D, NT, 1>(ring + out.slot * kHalf, q, key0, shown, s);
                    else
                        page_scores<D, NT, 2>(ring + out.slot * kHalf, q, key0, shown, s);
                }
                release();
                fill();
                alive = take();
                if (!alive) continue;
                if (shown != 0) {
                    if (mask == 0)
                        page_values<D, NT, 0>(ring + out.slot * kHalf, q, shown, s, st);
                    else
                        page_values<D, NT, 1>(ring + out.slot * kHalf, q, shown, s, st);
                }
                release();
                fill();
            }

            // ---- sums over the lanes that share a column
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) {
                        st.l[n][c] += __shfl_xor_sync(kFull, st.l[n][c], off);
#pragma unroll
                        for (int grp = 0; grp < G; ++grp) st.z[n][c][grp] += __shfl_xor_sync(kFull, st.z[n][c][grp], off);
                    }
                    // the maximum becomes the base of the weights, in log2 units
                    st.m[n][c] = st.l[n][c] > 0.0f ? fmaf(st.m[n][c], q.unit[n][c], static_cast<float>(st.e - kUp)) : kNegInf;
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            st.o[dt][n][2 * r + c] = fmaf(st.o[dt][n][2 * r + c], 0x1p24f, st.z[n][c][dt / 4]);
                }
            const bool whole = start == item.begin && flat == item.end;
            const bool last = flat == w1;
            if (whole) {
                store_item<D, NT, kSelected>(p, tile, item.head, group, st);
                continue;
            }
            // a partial result; the warp's last one takes the place of its
            // ring, which holds nothing more
            for (; last && alive && flight; release()) alive = take();
            float* part = last ? last_part(warp) : first_part(warp);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = n * 8 + 2 * t + c;
                    if (g == 0) {
                        part[kCols * (D + 4) + col] = st.m[n][c];
                        part[kCols * (D + 5) + col] = st.l[n][c];
                    }
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                        for (int r = 0; r < 2; ++r) part[col * (D + 4) + dt * 16 + 8 * r + g] = st.o[dt][n][2 * r + c];
                }
            if (lane == 0) mine.part[last ? 1 : 0] = item;
        }
        for (; alive && flight; release()) alive = take();
        if (!alive) {
            // what is still in flight may not outlive the block's shared memory
            for (; flight; release()) take();
            if (lane == 0) kv_timeout(batch);
        }
    }
    __syncthreads();

    // ---- join the warps' partial results of each item, in unit order: the
    // rows where the block has the whole item, else a partial result for the
    // joining kernel.  First the factors (a warp a column, a lane a partial
    // result), then the weighted sums.
    const auto part_of = [&](int e) -> const float* { return e & 1 ? last_part(e >> 1) : first_part(e >> 1); };
    const bool there = lane < 2 * kWarps && warp_items[lane >> 1].part[lane & 1].end != 0;
    const uint64_t begin = there ? warp_items[lane >> 1].part[lane & 1].begin : 0;
    unsigned left = __ballot_sync(kFull, there);  // entries still to be joined; the same in every warp
    while (left) {
        const int e0 = __ffs(left) - 1;
        const uint64_t first_begin = __shfl_sync(kFull, begin, e0);
        const unsigned mine_of = __ballot_sync(kFull, there && begin == first_begin) & left;
        left &= ~mine_of;
        const Item& item = warp_items[e0 >> 1].part[e0 & 1];
        const int cols = item.tile.cols;
        for (int c = warp; c < cols; c += kWarps) {
            const bool on = (mine_of >> lane) & 1;
            const float* part = part_of(on ? lane : e0);
            const float pm = on ? part[kCols * (D + 4) + c] : kNegInf;
            float m = pm;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, off));
            const float base = m == kNegInf ? 0.0f : m;
            const float f = on ? exp2_fast(pm - base) : 0.0f;
            float l = on ? part[kCols * (D + 5) + c] * f : 0.0f;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(kFull, l, off);
            factors[c * 32 + lane] = f;
            if (lane == 0) {
                factors[kCols * 32 + c] = m;
                factors[kCols * 33 + c] = l;
            }
        }
        __syncthreads();
        const bool whole = item.begin >= u0 && item.end <= u1;
        float* out_part = parts + (2ull * blockIdx.x + (item.begin <= u0 ? 0 : 1)) * kPartFloats<D, NT>;
        for (int i = threadIdx.x; i < cols * (D / 4); i += Cfg::kThreads) {
            const int c = i / (D / 4), d = i % (D / 4) * 4;
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (unsigned rest = mine_of; rest; rest &= rest - 1) {
                const int e = __ffs(rest) - 1;
                const float4 v = *reinterpret_cast<const float4*>(part_of(e) + c * (D + 4) + d);
                const float f = factors[c * 32 + e];
                o[0] = fmaf(v.x, f, o[0]);
                o[1] = fmaf(v.y, f, o[1]);
                o[2] = fmaf(v.z, f, o[2]);
                o[3] = fmaf(v.w, f, o[3]);
            }
            const float m = factors[kCols * 32 + c], l = factors[kCols * 33 + c];
            if (whole) {
                store_row<D>(p, item.tile, item.head, group, kSelected, c, d, m == kNegInf ? 0.0f : m, l, o);
            } else {
                if (d == 0) {
                    out_part[c] = m;
                    out_part[kCols + c] = l;
                }
                *reinterpret_cast<float4*>(out_part + 2 * kCols + c * D + d) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
        __syncthreads();
    }
}

// Items that several blocks share.  The factors of the partial results first,
// then their weighted sum in block order, all loads side by side; the sum does
// not depend on which block was done first.  Two dependent loads from L2 and a
// launch: 8 us under a profiler, about 5 behind the main kernel, which it is
// launched beside.
constexpr int kMaxBlocks = 192, kJoinThreads = 256;
template <int D, int NT, bool kSelected>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(gofann_kv_cache cache, gofann_kv_batch batch, Call p,
                                                               uint32_t blocks, const float* __restrict__ parts)
{
    constexpr int kCols = 8 * NT;
    __shared__ float factor[kMaxBlocks][kCols], total_of[kCols], base_of[kCols];
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const uint32_t n_kv = cache.n_kv_heads;
    // block i joins the item that the end of share i cuts, if that is the item's first cut
    uint64_t share = 0, cut = 0;
    SeqCursor c;
    const bool any = seek_by_total<kSelected>(
        batch, p, n_kv, group, kCols,
        [&](uint64_t total) {
            share = units_per_block(total, blocks, Attend<D, NT>::kWarps, 0);
            cut = share * (blockIdx.x + 1);
            return static_cast<unsigned long long>(cut < total ? cut : ~0ull);
        },
        c);
    if (!any) {
        wait_previous();
        return;
    }
    Item item;
    make_item<kSelected>(batch, p, n_kv, group, kCols, cut, c, item);
    if (item.begin >= cut || item.begin < share * blockIdx.x) {
        wait_previous();
        return;
    }
    const uint64_t first = blockIdx.x;
    const int count = static_cast<int>((item.end - 1) / share - first) + 1;
    const auto part_at = [&](int b) {
        return parts + (2 * (first + b) + (item.begin <= share * (first + b) ? 0 : 1)) * kPartFloats<D, NT>;
    };
    wait_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int col = warp; col < item.tile.cols; col += kJoinThreads / 32) {
        float m = kNegInf, l = 0.0f;
        for (int b = lane; b < count; b += 32) {
            const float x = __ldcg(part_at(b) + col);
            factor[b][col] = x;
            m = fmaxf(m, x);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, off));
        const float base = m == kNegInf ? 0.0f : m;
        for (int b = lane; b < count; b += 32) {
            const float f = exp2_fast(factor[b][col] - base);
            factor[b][col] = f;
            l = fmaf(__ldcg(part_at(b) + kCols + col), f, l);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(kFull, l, off);
        if (lane == 0) {
            base_of[col] = base;
            total_of[col] = l;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < item.tile.cols * (D / 4); i += kJoinThreads) {
        const int col = i / (D / 4), d = i % (D / 4) * 4;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int b = 0; b < count; ++b) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part_at(b) + 2 * kCols + col * D + d));
            const float f = factor[b][col];
            o[0] = fmaf(v.x, f, o[0]);
            o[1] = fmaf(v.y, f, o[1]);
            o[2] = fmaf(v.z, f, o[2]);
            o[3] = fmaf(v.w, f, o[3]);
        }
        store_row<D>(p, item.tile, item.head, group, kSelected, col, d, base_of[col], total_of[col], o);
    }
}

// The tensor memory kernel takes 256 query columns (rows x query heads of a
// key/value head) at a time, whatever there is of them; the other one's time
// grows with the columns.  8 sequences of 16384 tokens, 8 key/value heads, us
// (the other kernel / tensor memory): head_dim 128 at 64 columns 190 / 260, at
// 128 326 / 272, at 256 601 / 292; head_dim 64 at 128 columns 190 / 202, at 256
// 352 / 215.
constexpr uint64_t kManyColumnDims = 128 * 128;
bool many_columns(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p)
{
    return !p.selected && cache.n_kv_heads &&
           static_cast<uint64_t>(batch.max_rows) * (p.n_heads / cache.n_kv_heads) * cache.head_dim >= kManyColumnDims;
}

// Cache blocks that an item can have at most.
uint64_t most_blocks(const gofann_kv_batch& batch, const gofann_kv_attention_params& p)
{
    const uint64_t span = p.selected ? p.n_select : batch.max_pages;
    return span ? span : 1;
}

// Thread blocks of the attention kernel: one per SM (the ring takes most of
// its shared memory), no more than there can be units (items, where each is
// done by one block).
uint32_t attend_blocks(const gofann_kv_batch& batch, const Call& p)
{
    const uint64_t most = static_cast<uint64_t>(batch.n_rows) * p.n_heads * (p.fixed ? 1 : most_blocks(batch, p));
    const int sms = sm_count() < kMaxBlocks ? sm_count() : kMaxBlocks;
    const uint64_t want = sms > 0 ? sms : 1;
    return static_cast<uint32_t>(most < want ? most : want);
}

template <int D, int NT, bool kSelected>
int launch_attend(const gofann_kv_cache& cache, const gofann_kv_batch& batch, Call p, float* parts, cudaStream_t s)
{
    using Cfg = Attend<D, NT>;
    // Items of at most two pages a warp stay in one block: what a split would
    // gain, the joining kernel would cost (one row over 777 tokens 12.6 us, split
    // 16.5; 509 rows of 32 selected blocks 86 us, split 90).
    p.fixed = most_blocks(batch, p) <= 2 * Cfg::kWarps ? static_cast<int>(most_blocks(batch, p)) : 0;
    auto* kernel = kv_attend_kernel<D, NT, kSelected>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg::kBytes));
    if (e != cudaSuccess) return cuda_status(e, "kv_attention: shared memory attribute");
    const uintptr_t q = reinterpret_cast<uintptr_t>(p.q);
    const bool wide = (q & 7) == 0 && (p.q_stride & 3) == 0;
    const uint32_t blocks = attend_blocks(batch, p);
    kernel<<<blocks, Cfg::kThreads, Cfg::kBytes, s>>>(cache, batch, p, wide, parts);
    GOFANN_CHECK_LAUNCH("kv_attend_kernel");
    if (blocks == 1 || p.fixed) return GOFANN_OK;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks - 1);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv_join_kernel<D, NT, kSelected>, cache, batch, p, blocks, static_cast<const float*>(parts));
    if (e != cudaSuccess) return cuda_status(e, "kv_join_kernel");
    return GOFANN_OK;
}

}  // namespace
}  // namespace gofann

using namespace gofann;

extern "C" {

size_t gofann_kv_attention_scratch_bytes(const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                                         const gofann_kv_attention_params* params)
{
    if (!cache || !batch || !params) return 0;
    const size_t part = sizeof(float) * (cache->head_dim <= 64 ? kPartFloats<64, 2> : kPartFloats<128, 2>);
    const int sms = sm_count() > 0 ? sm_count() : 1;
    if (many_columns(*cache, *batch, *params)) return attend_rows_scratch(cache->head_dim, sms);
    return 2 * part * static_cast<size_t>(sms);
}

int gofann_kv_attention(const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                        const gofann_kv_attention_params* params, void* scratch, size_t scratch_bytes, void* stream)
{
    if (!params) return fail(GOFANN_ERR_INVALID, "kv_attention: null descriptor");
    Call p;
    static_cast<gofann_kv_attention_params&>(p) = *params;
    p.fixed = 0;
    int st = kv_check("kv_attention", cache, batch, p.dtype, p.n_heads);
    if (st != GOFANN_OK) return st;
    const uint32_t d = cache->head_dim;
    if (!(p.scale > kNegInf && p.scale < -kNegInf)) return fail(GOFANN_ERR_INVALID, "kv_attention: scale is not finite");
    if (p.selected && p.n_select == 0) return fail(GOFANN_ERR_INVALID, "kv_attention: selected of width 0");
    if (p.n_select > 0x7fffffffu) return fail(GOFANN_ERR_UNSUPPORTED, "kv_attention: n_select %u", p.n_select);
    if (batch->n_rows == 0) return GOFANN_OK;
    if (!p.q || !p.out) return fail(GOFANN_ERR_INVALID, "kv_attention: null queries or output");
    if (!cache->pages || batch->max_pages == 0) return fail(GOFANN_ERR_INVALID, "kv_attention: rows without pages");
    if (p.q_stride < static_cast<uint64_t>(p.n_heads) * d)
        return fail(GOFANN_ERR_INVALID, "kv_attention: a row stride is shorter than its row");
    auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    if ((bits(cache->pages) & 15) || (bits(p.out) & 7) || (bits(p.q) & 1))
        return fail(GOFANN_ERR_INVALID, "kv_attention: pages must be 16-byte, out 8-byte, queries 2-byte aligned");
    const size_t need = gofann_kv_attention_scratch_bytes(cache, batch, params);
    if (!scratch || (bits(scratch) & 255)) return fail(GOFANN_ERR_INVALID, "kv_attention: scratch must be 256-byte aligned");
    if (scratch_bytes < need)
        return fail(GOFANN_ERR_CAPACITY, "kv_attention: scratch of %zu bytes, %zu needed", scratch_bytes, need);
    const uint32_t group = p.n_heads / cache->n_kv_heads;
    const uint64_t cols = p.selected ? group : static_cast<uint64_t>(batch->max_rows) * group;
    cudaStream_t s = as_stream(stream);
    float* parts = static_cast<float*>(scratch);
    if (many_columns(*cache, *batch, p)) return attend_rows(*cache, *batch, p, parts, s);
#define GOFANN_KV_LAUNCH(D, NT)                                                   \
    return p.selected ? launch_attend<D, NT, true>(*cache, *batch, p, parts, s) \
                      : launch_attend<D, NT, false>(*cache, *batch, p, parts, s)
    if (d == 64) {
        if (cols <= 8) GOFANN_KV_LAUNCH(64, 1);
        GOFANN_KV_LAUNCH(64, 2);
    }
    if (cols <= 8) GOFANN_KV_LAUNCH(128, 1);
    GOFANN_KV_LAUNCH(128, 2);
#undef GOFANN_KV_LAUNCH
}

}  // extern "C"
