// kv_attention.cu — attention over the 4-bit cache.
//
// With codes c, scales s and minima m (per token and 64 dimensions),
//   q.k   = sum_grp s_grp (q_grp . c_grp) + m_grp (sum of q_grp)
//   sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)
// so the matrix instructions read the codes themselves.  A code word masked
// to nibbles is already a pair of f16 numbers: 0x000c is the subnormal
// c * 2^-24 and 0x00c0 is c * 2^-20, both exact, so two ANDs and a shift turn
// 32 bits into half of an A operand.  The 2^-24 goes into the f32 scale, the
// extra 2^4 of the odd nibbles into the other operand.
//
// Tokens are the rows (M = 16) and query heads the columns (N = 8) of both
// products: S^T = K Q^T, then O^T = V^T P^T; the transposition of P between
// the two layouts is one movmatrix per 8 x 8 tile.
#include "kv_async.cuh"

namespace gofann {
namespace {

constexpr int kAttendThreads = 256;
constexpr int kAttendWarps = kAttendThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 2^x by the special function unit (2 ulp; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
__device__ __forceinline__ float low_half(uint32_t w)
{
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu)));
}
__device__ __forceinline__ float high_half(uint32_t w)
{
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
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

// The query columns that a block works on at a time: rows of a sequence x
// query heads of one key/value head, and the cache blocks that any of them
// sees.
struct Tile {
    uint32_t seq;
    int first_row, n_rows, len;  // of the sequence
    int col0, cols;              // columns of the sequence (dense) or of the row (selected)
    int row;                     // selected: the row inside the sequence
    int block_lo, block_hi;      // cache blocks (dense) or slots of the list (selected)
};

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

// A sequence's share of the work in units of one cache block for one tile and
// key/value head: every tile counts `span` blocks from `lo` on (what all of
// the sequence's rows see), at least one, so that each tile has an owner.
struct SeqWork {
    int tiles, lo, span;
};
template <bool kSelected>
__device__ __forceinline__ SeqWork seq_work(const gofann_kv_batch& b, const gofann_kv_attention_params& p, int group,
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
    w.span = hi > lo ? hi - lo : 1;
    return w;
}

// Blocks [b0, b1) of one tile and head, and its place among all units.
struct Segment {
    Tile tile;
    uint32_t head;
    int b0, b1;
    uint64_t item_begin, item_end, end;  // units of the whole (tile, head), and where this part ends
};

template <bool kSelected>
__device__ __forceinline__ void make_tile(const gofann_kv_batch& b, const gofann_kv_attention_params& p, int group,
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
        tile.block_lo = 0;
        tile.block_hi = static_cast<int>(p.n_select);
    } else {
        const int total = tile.n_rows * group;
        tile.row = 0;
        tile.col0 = at * width;
        tile.cols = total - tile.col0 < width ? total - tile.col0 : width;
        dense_blocks(p, group, tile.len, tile.n_rows, tile.col0, tile.cols, tile.block_lo, tile.block_hi);
    }
}

// The segment of units [flat, limit) that starts at `flat`; false at the end.
template <bool kSelected>
__device__ __forceinline__ bool segment_at(const gofann_kv_batch& b, const gofann_kv_attention_params& p, uint32_t n_kv,
                                           int group, int width, uint64_t flat, uint64_t limit, Segment& sg)
{
    if (flat >= limit) return false;
    uint32_t seq;
    uint64_t at;
    const auto units = [&](uint32_t s) {
        const SeqWork w = seq_work<kSelected>(b, p, group, width, s);
        return static_cast<uint64_t>(w.tiles) * n_kv * w.span;
    };
    if (!kv_find<uint64_t>(b.n_seqs, flat, units, seq, at)) return false;
    const SeqWork w = seq_work<kSelected>(b, p, group, width, seq);
    const uint64_t item = at / w.span;
    const int off = static_cast<int>(at % w.span);
    sg.head = static_cast<uint32_t>(item % n_kv);
    make_tile<kSelected>(b, p, group, width, seq, static_cast<int>(item / n_kv), sg.tile);
    sg.item_begin = flat - off;
    sg.item_end = sg.item_begin + w.span;
    sg.end = sg.item_end < limit ? sg.item_end : limit;
    const int b0 = w.lo + off, b1 = w.lo + static_cast<int>(sg.end - sg.item_begin);
    sg.b0 = b0 > sg.tile.block_lo ? b0 : sg.tile.block_lo;
    sg.b1 = b1 < sg.tile.block_hi ? b1 : sg.tile.block_hi;
    return true;
}

// Running softmax state of one warp: columns 2t, 2t + 1 of each 8-column
// tile, dimensions 16 dt + g, + 8.
template <int D, int NT>
struct State {
    float m[NT][2], l[NT][2];            // max (log2 units) and this lane's part of the sum
    float z[NT][2][KvChunk<D>::kGroups]; // this lane's part of sum p * (minimum + 8 scale)
    float o[D / 16][NT][4];              // sum (p * scale * 2^(26 - e)) * (code - 8) * 2^-24
    int e;                               // largest exponent of a value scale so far
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

// The query columns as B operands and their f32 companions.
template <int D, int NT>
struct Query {
    uint32_t b[D / 16][NT][2];
    float scale[NT][2];                        // logits in log2 units per unit of the product with codes
    float sum[NT][2][KvChunk<D>::kGroups];     // sum of the column over a group, in log2 units
    int limit[NT][2], low[NT][2];              // keys seen: low < key <= limit
};

// One page: scores, softmax update, weighted values.  `masked`: some token
// of the page is hidden from some column; `shown` has a bit per token.
template <int D, int NT>
__device__ __forceinline__ void attend_page(const unsigned char* chunk, const Query<D, NT>& q, State<D, NT>& st,
                                            int key0, bool masked, uint64_t shown)
{
    using Chunk = KvChunk<D>;
    constexpr int G = Chunk::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const int first = 16 * (g >> 1) + (g & 1);  // this lane's tokens: first + 2 i, i = 0 .. 7
    float s[4][NT][4];

    // ---- scores of 64 tokens x 8 NT columns
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kt][n][i] = 0.0f;
        uint32_t kp[2 * G];  // tokens first + 4 kt, + 2
        load_words<2 * G>(chunk + Chunk::kKeyParams + (g * 4 + kt) * 8 * G, kp);
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            const uint4 w4 = reinterpret_cast<const uint4*>(chunk)[(kt * G + grp) * 32 + lane];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a[4];
                code_operand(w[j], a);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(acc[n], a, q.b[grp * 4 + j][n][0], q.b[grp * 4 + j][n][1]);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float ks = low_half(kp[r * G + grp]), km = high_half(kp[r * G + grp]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        s[kt][n][2 * r + c] += fmaf(acc[n][2 * r + c] * q.scale[n][c], ks, km * q.sum[n][c][grp]);
            }
        }
    }
    if (masked) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int token = first + 4 * kt + 2 * r, key = key0 + token;
                const bool on = (shown >> token) & 1;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        if (!on || key > q.limit[n][c] || key <= q.low[n][c]) s[kt][n][2 * r + c] = kNegInf;
            }
    }

    // ---- the largest value scale; a hidden token's params may be anything,
    // so they count as 0 here and below
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t w[G];
        load_words<G>(chunk + Chunk::kValueParams + (g * 8 + i) * 4 * G, w);
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
            if (!masked || ((shown >> (first + 2 * i)) & 1)) top = max(top, w[grp] & 0x7c00u);
    }
    // The weights p * scale become f16 operands.  They are taken relative to
    // the largest scale exponent so far (2^26-e below), so that f16 holds
    // them from 2^12 down to 2^-24 whatever the values' magnitude.
    const int e = max(st.e, static_cast<int>(__reduce_max_sync(kFull, top) >> 10));
    float rescale[NT][2];
    const float shift = exp2f(static_cast<float>(st.e - e));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float mx = st.m[n][c];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) mx = fmaxf(mx, fmaxf(s[kt][n][c], s[kt][n][2 + c]));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
            const float use = mx == kNegInf ? 0.0f : mx;
            const float f = exp2_fast(st.m[n][c] - use);
            st.m[n][c] = mx;
            st.l[n][c] *= f;
#pragma unroll
            for (int grp = 0; grp < G; ++grp) st.z[n][c][grp] *= f;
            rescale[n][c] = f * shift;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x = exp2_fast(s[kt][n][2 * r + c] - use);
                    s[kt][n][2 * r + c] = x;
                    st.l[n][c] += x;
                }
        }
    st.e = e;

    // ---- weighted values.  The matrix instruction truncates its sums, so a
    // long chain of the codes' one-sided products would drift: codes are
    // centred (8 times the sum of the weights is taken off by the same
    // instructions on a constant operand) and a page's sum joins the running
    // one by an f32 fma that also rescales it.
    const uint32_t eight[4] = {0x80088008u, 0x80088008u, 0x80808080u, 0x80808080u};  // -8 * 2^-24, -8 * 2^-20
    const float up = exp2f(static_cast<float>(26 - e));
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
        uint32_t b[4][NT][2];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                uint32_t w = reinterpret_cast<const uint32_t*>(chunk + Chunk::kValueParams)[(g * 8 + 2 * kt + r) * G + grp];
                if (masked && !((shown >> (first + 4 * kt + 2 * r)) & 1)) w = 0;
                const float scale = low_half(w), vs = scale * (r ? up * 0.0625f : up);
                const float vm = fmaf(8.0f, scale, high_half(w));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float p0 = s[kt][n][2 * r], p1 = s[kt][n][2 * r + 1];
                    st.z[n][0][grp] = fmaf(p0, vm, st.z[n][0][grp]);
                    st.z[n][1][grp] = fmaf(p1, vm, st.z[n][1][grp]);
                    b[kt][n][r] = transpose8x8(pack_f16(p0 * vs, p1 * vs));
                }
            }
        float centre[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) centre[n][i] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) mma_f16(centre[n], eight, b[kt][n][0], b[kt][n][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dt = grp * 4 + i;
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[n][k] = centre[n][k];
            const uint4 w4 = reinterpret_cast<const uint4*>(chunk + Chunk::kValueCodes)[dt * 32 + lane];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t a[4];
                code_operand(w[kt], a);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(acc[n], a, b[kt][n][0], b[kt][n][1]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) st.o[dt][n][k] = fmaf(st.o[dt][n][k], rescale[n][k & 1], acc[n][k]);
        }
    }
}

template <int D, int NT>
__device__ __forceinline__ void load_query(const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                                           const Tile& tile, uint32_t head, int group, bool selected, bool wide,
                                           Query<D, NT>& q)
{
    constexpr int G = KvChunk<D>::kGroups;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
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
        float sum[G];
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            sum[grp] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    top = fmaxf(top, fabsf(x[grp][j][k]));
                    sum[grp] += x[grp][j][k];
                }
            sum[grp] += __shfl_xor_sync(kFull, sum[grp], 1);
            sum[grp] += __shfl_xor_sync(kFull, sum[grp], 2);
        }
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
        // a power of two brings the column's largest value to [2^13, 2^14):
        // every bf16 or f16 within 2^27 of it is then an exact f16
        int ex = static_cast<int>(__float_as_uint(top) >> 23);
        ex = ex < 28 ? 28 : ex > 240 ? 240 : ex;
        const float down = __uint_as_float(static_cast<uint32_t>(267 - ex) << 23);  // 2^(140 - ex)
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float(&y)[4] = x[grp][j];
                q.b[grp * 4 + j][n][0] = pack_f16(y[0] * down, y[1] * down);
                q.b[grp * 4 + j][n][1] = pack_f16(y[2] * down * 0.0625f, y[3] * down * 0.0625f);
            }
        const float unit = p.scale * kLog2e;
        // 2^(ex - 140) undoes `down`, 2^24 the codes' subnormals
        const float undo = unit * exp2f(static_cast<float>(ex - 140 + 24));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            q.scale[n][e] = __shfl_sync(kFull, undo, 4 * (2 * t + e));
#pragma unroll
            for (int grp = 0; grp < G; ++grp) q.sum[n][e][grp] = __shfl_sync(kFull, sum[grp] * unit, 4 * (2 * t + e));
            const int cc = n * 8 + 2 * t + e;
            const int row = selected ? tile.row : (tile.col0 + cc) / group;
            const int pos = tile.len - tile.n_rows + row;
            // padding columns see what the tile's last column sees
            int limit = p.causal ? (pos < tile.len ? pos : tile.len - 1) : tile.len - 1;
            if (pos < 0) limit = -1;
            const long long low = p.window ? static_cast<long long>(pos) - p.window : -1;
            q.limit[n][e] = limit;
            q.low[n][e] = low > -1 ? static_cast<int>(low) : -1;
            if (cc >= tile.cols) {  // no mask of its own: nothing of it is written
                q.limit[n][e] = 0x7fffffff;
                q.low[n][e] = -1;
            }
        }
    }
}

// Shared memory of a block: a ring of kStages chunks per warp, the warps'
// partial results of a segment, the ring's barriers.
template <int D, int NT>
struct AttendShared {
    static constexpr int kCols = 8 * NT;
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr size_t kRing = static_cast<size_t>(kAttendWarps) * kStages * KvChunk<D>::kBytes;
    static constexpr size_t kMerge = sizeof(float) * kAttendWarps * kCols * (D + 4 + 2);
    static constexpr size_t kBytes = kRing + kMerge + sizeof(uint64_t) * kAttendWarps * kStages;
};

// Units of one block: a share of the total, at least one per warp.
__device__ __forceinline__ uint64_t units_per_block(uint64_t total, uint32_t blocks)
{
    const uint64_t c = (total + blocks - 1) / blocks;
    return c > kAttendWarps ? c : kAttendWarps;
}

// A partial result in scratch: [cols] max, [cols] sum, [cols][D] values; two
// per block (its first segment, and its last if that is another).
template <int D, int NT>
constexpr size_t kPartFloats = 8 * NT * (D + 2);

template <int D>
__device__ __forceinline__ void store_row(const gofann_kv_attention_params& p, const Tile& tile, uint32_t head, int group,
                                          bool selected, int c, int d, float m, float l, const float (&o)[4])
{
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int col = tile.col0 + c;
    const uint64_t row = tile.first_row + (selected ? tile.row : col / group);
    const uint64_t at = row * p.n_heads + head * group + (selected ? col : col % group);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * D + d) =
        l > 0.0f ? make_uint2(kv_pack2(o[0] * inv, o[1] * inv, p.dtype), kv_pack2(o[2] * inv, o[3] * inv, p.dtype))
                 : make_uint2(0u, 0u);
    if (d == 0 && p.lse) p.lse[at] = l > 0.0f ? (m + log2f(l)) * kLn2 : kNegInf;
}

// The chunks that a warp reads, in order: its share (every kAttendWarps-th
// block) of each segment of the thread block.  Page numbers are looked up 32
// blocks at a time, one per lane.
template <int D, bool kSelected>
struct Reader {
    Segment sg;
    int next;       // this warp's next block (or slot) of the segment
    int batch_at;   // `next` of lane 0's entry
    int block, page;  // this lane's entry: cache block and page, -1 = nothing to read
    bool more;

    __device__ __forceinline__ void look_up(const gofann_kv_cache& cache, const gofann_kv_batch& b,
                                            const gofann_kv_attention_params& p)
    {
        const int lane = threadIdx.x & 31;
        const int i = next + lane * kAttendWarps;
        batch_at = next;
        block = page = -1;
        if (i < sg.b1) {
            const int seq_blocks = (sg.tile.len + kKvPage - 1) / kKvPage;
            block = i;
            if (kSelected)
                block = __ldg(p.selected +
                              (static_cast<size_t>(sg.tile.first_row + sg.tile.row) * cache.n_kv_heads + sg.head) * p.n_select + i);
            if (block >= 0 && block < seq_blocks) {
                page = __ldg(b.page_table + static_cast<size_t>(sg.tile.seq) * b.max_pages + block);
                if (page < 0 || static_cast<uint32_t>(page) >= cache.n_pages) {
                    page = -1;
                    kv_invalid(b);
                }
            }
        }
    }
};

template <int D, int NT, bool kSelected>
__global__ void __launch_bounds__(kAttendThreads, 1) kv_attend_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                                      gofann_kv_attention_params p, bool wide,
                                                                      float* __restrict__ parts)
{
    using Chunk = KvChunk<D>;
    using Shared = AttendShared<D, NT>;
    constexpr int G = Chunk::kGroups, kCols = 8 * NT, kStages = Shared::kStages;
    extern __shared__ __align__(128) unsigned char smem[];
    float* merge_o = reinterpret_cast<float*>(smem + Shared::kRing);  // [warps][cols][D + 4]
    float* merge_m = merge_o + kAttendWarps * kCols * (D + 4);        // [warps][cols]
    float* merge_l = merge_m + kAttendWarps * kCols;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const unsigned char* ring = smem + static_cast<size_t>(warp) * kStages * Chunk::kBytes;
    const uint32_t bars = shared_addr(smem + Shared::kRing + Shared::kMerge) + warp * kStages * 8;
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);

    if (lane < kStages) barrier_init(bars + 8 * lane, 1);
    barrier_fence();
    launch_next();
    __syncwarp();
    const auto units = [&](uint32_t s) {
        const SeqWork w = seq_work<kSelected>(batch, p, group, kCols, s);
        return static_cast<uint64_t>(w.tiles) * cache.n_kv_heads * w.span;
    };
    const uint64_t total = kv_total<uint64_t>(batch.n_seqs, units);
    const uint64_t share = units_per_block(total, gridDim.x);
    const uint64_t u0 = share * blockIdx.x, u1 = u0 + share < total ? u0 + share : total;
    if (u0 >= u1) return;

    // ---- the loads run ahead of the work by up to kStages chunks
    Reader<D, kSelected> rd;
    rd.more = segment_at<kSelected>(batch, p, cache.n_kv_heads, group, kCols, u0, u1, rd.sg);
    rd.next = rd.sg.b0 + warp;
    rd.look_up(cache, batch, p);
    uint32_t issued = 0, taken = 0;  // chunks of this warp
    const auto advance = [&]() {     // issues the next chunk's load, skipping entries with nothing to read
        while (rd.more) {
            if (rd.next >= rd.sg.b1) {
                rd.more = segment_at<kSelected>(batch, p, cache.n_kv_heads, group, kCols, rd.sg.end, u1, rd.sg);
                if (!rd.more) return;
                rd.next = rd.sg.b0 + warp;
                rd.look_up(cache, batch, p);
                continue;
            }
            int l = (rd.next - rd.batch_at) / kAttendWarps;
            if (l >= 32) {
                rd.look_up(cache, batch, p);
                l = 0;
            }
            const int page = __shfl_sync(kFull, rd.page, l);
            rd.next += kAttendWarps;
            if (page < 0) continue;
            if (lane == 0) {
                const uint32_t st = issued % kStages;
                barrier_expect(bars + 8 * st, Chunk::kBytes);
                bulk_load(shared_addr(ring + st * Chunk::kBytes),
                          cache.pages + (static_cast<size_t>(page) * cache.n_kv_heads + rd.sg.head) * Chunk::kBytes,
                          Chunk::kBytes, bars + 8 * st);
            }
            ++issued;
            return;
        }
    };
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) advance();

    // ---- segment by segment
    bool alive = true;  // false once a wait has run out
    uint64_t flat = u0;
    Reader<D, kSelected> use;
    while (segment_at<kSelected>(batch, p, cache.n_kv_heads, group, kCols, flat, u1, use.sg)) {
        const Segment& sg = use.sg;
        const Tile& tile = sg.tile;
        Query<D, NT> q;
        load_query<D, NT>(batch, p, tile, sg.head, group, kSelected, wide, q);
        int limit = 0x7fffffff, low = -1;  // keys in (low, limit] are seen by every column
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                limit = min(limit, q.limit[n][e]);
                low = max(low, q.low[n][e]);
            }
        limit = __reduce_min_sync(kFull, limit);
        low = __reduce_max_sync(kFull, low);
        State<D, NT> st;
        clear(st);
        use.next = sg.b0 + warp;
        while (use.next < sg.b1) {
            use.look_up(cache, batch, p);
            const uint32_t* bits = p.key_bits ? p.key_bits + static_cast<size_t>(tile.seq) * p.key_words : nullptr;
#pragma unroll 1
            for (int l = 0; l < 32 && use.next < sg.b1; ++l, use.next += kAttendWarps) {
                if (__shfl_sync(kFull, use.page, l) < 0) continue;
                const int block = __shfl_sync(kFull, use.block, l), key0 = block * kKvPage;
                uint64_t shown = ~0ull;
                if (bits) {
                    const uint32_t w = 2u * block;
                    shown = (w < p.key_words ? __ldg(bits + w) : 0u) |
                            (static_cast<uint64_t>(w + 1 < p.key_words ? __ldg(bits + w + 1) : 0u) << 32);
                }
                if (tile.len - key0 < kKvPage) shown &= (1ull << (tile.len - key0)) - 1;
                const bool masked = shown != ~0ull || key0 + kKvPage - 1 > limit || key0 <= low;
                const uint32_t stage = taken % kStages;
                alive = alive && barrier_wait(bars + 8 * stage, (taken / kStages) & 1);
                if (!alive) continue;
                attend_page<D, NT>(ring + stage * Chunk::kBytes, q, st, key0, masked, shown);
                ++taken;
                __syncwarp();
                advance();
            }
        }

        // ---- this warp's partial result, in units of its own maximum
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = n * 8 + 2 * t + c;
                float l = st.l[n][c];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(kFull, l, off);
                if (g == 0) {
                    merge_m[warp * kCols + col] = st.m[n][c];
                    merge_l[warp * kCols + col] = l;
                }
                const float unit = exp2f(static_cast<float>(st.e - 2));  // 2^24 of the codes, 2^(e - 26) of the weights
#pragma unroll
                for (int grp = 0; grp < G; ++grp) {
                    float z = st.z[n][c][grp];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) z += __shfl_xor_sync(kFull, z, off);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            merge_o[(warp * kCols + col) * (D + 4) + (grp * 4 + i) * 16 + 8 * r + g] =
                                fmaf(st.o[grp * 4 + i][n][2 * r + c], unit, z);
                }
            }
        __syncthreads();

        // ---- join the warps: the output where the block has the whole item,
        // else a partial result for the joining kernel
        const bool whole = flat == sg.item_begin && sg.end == sg.item_end;
        float* part = parts + (2ull * blockIdx.x + (flat == u0 ? 0 : 1)) * kPartFloats<D, NT>;
        for (int i = threadIdx.x; i < tile.cols * (D / 4); i += kAttendThreads) {
            const int c = i / (D / 4), d = i % (D / 4) * 4;
            float m = kNegInf;
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, merge_m[w * kCols + c]);
            float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) {
                const float f = exp2_fast(merge_m[w * kCols + c] - base);
                const float4 v = *reinterpret_cast<const float4*>(&merge_o[(w * kCols + c) * (D + 4) + d]);
                l = fmaf(merge_l[w * kCols + c], f, l);
                o[0] = fmaf(v.x, f, o[0]);
                o[1] = fmaf(v.y, f, o[1]);
                o[2] = fmaf(v.z, f, o[2]);
                o[3] = fmaf(v.w, f, o[3]);
            }
            if (whole) {
                store_row<D>(p, tile, sg.head, group, kSelected, c, d, m, l, o);
            } else {
                if (d == 0) {
                    part[c] = m;
                    part[kCols + c] = l;
                }
                *reinterpret_cast<float4*>(part + 2 * kCols + c * D + d) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
        __syncthreads();
        flat = sg.end;
    }
    // loads in flight may not outlive the block's shared memory
    for (; taken < issued; ++taken) alive = barrier_wait(bars + 8 * (taken % kStages), (taken / kStages) & 1) && alive;
    if (!alive && lane == 0) kv_timeout(batch);
}

// Items that several blocks share: their partial results in block order, so
// that the sum does not depend on which block was done first.
template <int D, int NT, bool kSelected>
__global__ void __launch_bounds__(128) kv_join_kernel(gofann_kv_cache cache, gofann_kv_batch batch,
                                                      gofann_kv_attention_params p, uint32_t blocks,
                                                      const float* __restrict__ parts)
{
    constexpr int kCols = 8 * NT;
    const int group = static_cast<int>(p.n_heads / cache.n_kv_heads);
    const auto units = [&](uint32_t s) {
        const SeqWork w = seq_work<kSelected>(batch, p, group, kCols, s);
        return static_cast<uint64_t>(w.tiles) * cache.n_kv_heads * w.span;
    };
    const uint64_t share = units_per_block(kv_total<uint64_t>(batch.n_seqs, units), blocks);
    // the blocks' ends inside items: block i joins the item that end i falls into, if it is the item's first
    const uint64_t cut = share * (blockIdx.x + 1);
    Segment sg;
    if (!segment_at<kSelected>(batch, p, cache.n_kv_heads, group, kCols, cut, ~0ull, sg)) return;
    if (sg.item_begin >= cut || sg.item_begin < share * blockIdx.x) return;
    wait_previous();
    const uint64_t first = blockIdx.x, last = (sg.item_end - 1) / share;
    for (int i = threadIdx.x; i < sg.tile.cols * (D / 4); i += 128) {
        const int c = i / (D / 4), d = i % (D / 4) * 4;
        float m = kNegInf, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint64_t b = first; b <= last; ++b) {
            const bool start = share * b >= sg.item_begin;  // the item is the block's first segment
            const float* part = parts + (2 * b + (start ? 0 : 1)) * kPartFloats<D, NT>;
            const float pm = __ldcg(part + c), pl = __ldcg(part + kCols + c);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part + 2 * kCols + c * D + d));
            const float top = fmaxf(m, pm), base = top == kNegInf ? 0.0f : top;
            const float f = exp2_fast(m - base), h = exp2_fast(pm - base);
            l = l * f + pl * h;
            o[0] = o[0] * f + v.x * h;
            o[1] = o[1] * f + v.y * h;
            o[2] = o[2] * f + v.z * h;
            o[3] = o[3] * f + v.w * h;
            m = top;
        }
        store_row<D>(p, sg.tile, sg.head, group, kSelected, c, d, m, l, o);
    }
}

// Thread blocks of the attention kernel: one per SM (the ring takes most of
// its shared memory), no more than there can be units.
uint32_t attend_blocks(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p)
{
    const uint64_t span = p.selected ? p.n_select : batch.max_pages;
    const uint64_t units = static_cast<uint64_t>(batch.n_rows) * p.n_heads * (span ? span : 1);
    const uint64_t most = (units + kAttendWarps - 1) / kAttendWarps;
    const int sms = sm_count();
    const uint64_t want = sms > 0 ? sms : 1;
    return static_cast<uint32_t>(most < want ? most : want);
}

template <int D, int NT, bool kSelected>
int launch_attend(const gofann_kv_cache& cache, const gofann_kv_batch& batch, const gofann_kv_attention_params& p,
                  float* parts, cudaStream_t s)
{
    const size_t smem = AttendShared<D, NT>::kBytes;
    auto* kernel = kv_attend_kernel<D, NT, kSelected>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return cuda_status(e, "kv_attention: shared memory attribute");
    const uintptr_t q = reinterpret_cast<uintptr_t>(p.q);
    const bool wide = (q & 7) == 0 && (p.q_stride & 3) == 0;
    const uint32_t blocks = attend_blocks(cache, batch, p);
    kernel<<<blocks, kAttendThreads, smem, s>>>(cache, batch, p, wide, parts);
    GOFANN_CHECK_LAUNCH("kv_attend_kernel");
    if (blocks == 1) return GOFANN_OK;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks - 1);
    cfg.blockDim = dim3(128);
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
    const int sms = sm_count();
    return 2 * part * static_cast<size_t>(sms > 0 ? sms : 1);
}

int gofann_kv_attention(const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                        const gofann_kv_attention_params* params, void* scratch, size_t scratch_bytes, void* stream)
{
    if (!params) return fail(GOFANN_ERR_INVALID, "kv_attention: null descriptor");
    const gofann_kv_attention_params& p = *params;
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
