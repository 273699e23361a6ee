// Softmax cross entropy of an output head, x . W^T over a large vocabulary, and its gradient, in pieces of the vocabulary: the logits are
// never kept whole (but those of few tokens in fp32); of their gradient there are two pieces at a time.
//
//   lse[t] = log sum_v exp <x_t, w_v>,  nll[t] = lse[t] - <x_t, w_target[t]>,  loss = their mean, their sum, or nll itself
//   G[t][v] = (exp(<x_t, w_v> - lse[t]) - [v == target[t]]) g_t,   dx = G . W,   dW = G^T . x
//
// What rows hold whose target is the ignored label, NaN included, reaches no sum: they are read and left out before anything is multiplied (head_gather_kernel); up to 64 tokens of a
// forward call, and in the products of fp32, they are multiplied with the others and left out behind that.  A target outside the classes makes its row NaN.
//
// On the tiles of rdb_duo.hpp (bf16; of few tokens on those of rdb_gemm.hpp; fp32 in three bf16 planes, where that is faster):
//   head_gather_kernel      the rows that count, one after the other, in rows of a multiple of 8 values
//   head_logits_duo_kernel  a tile of logits in the accumulators -> its maximum and its sum of exponentials for each token, and the target's logit; or (backward), a piece
//   head_logits_solo_kernel of the vocabulary's logits once more -> G, in bf16, for the next launch
//   head_logits_few_kernel  (all tokens in one tile)
//   head_merge_kernel       the tiles of a token together, nll; the last block adds up the tokens
//   head_products_kernel    dx += G . W and dW = G^T . x of the piece, and the next piece's G, one list of tiles
//   head_dx_kernel          dx from its sums, back in the rows' own places
// G leaves without the factor that all its rows share (1 / count, the loss's gradient), which the products' results get in fp32: rounded with it, the targets' values,
// which are nearly all of the gradient, would all be off by the same rounding.  G in 16 bits is a choice: two planes of it would double two of four products.  dx and dW are 1.9e-3 - 2.0e-3 of their norms
// from 64 bits with it, 2.2e-3 where rows have factors of their own, which are in G; their own rounding alone is 1.7e-3.
// fp32 otherwise: the products of rdb_f32.hip, or of few tokens head_few_*_kernel, logits of a piece in fp32 in between, which of few tokens stay for the
// backward pass (rdb_linear_cross_entropy_keeps); ignored rows are rows of zeros of G there.
//
// Bound by the matrix cores, and these by their power: with 1 - 2 us of their own behind every tile hidden (two blocks a compute unit) the matrix cores are busy 66 % of the time at
// 1.65 GHz in the statistics and 58 - 65 % at 1.75 - 1.8 GHz in the products (8192 tokens x 768 -> 50304).  Requesting a block's next tile before its epilogue, other orders of the tiles and a higher
// priority for the main loop all change nothing.  Measured there, us: statistics 550 - 680, by the card (1150 - 930 TFLOP/s; the library's product alone 656), backward 1700 (three
// products, 1900 GFLOP), a step 2330; 8192 x 256 -> 50304 1060; 4096 x 4096 -> 65536 7080 (four products, 1240 TFLOP/s).
#include "rdb_duo.hpp"
#include "rdb_f32.hpp"
#include <algorithm>

namespace rdb {

int num_compute_units();
int f32_split_mode();

constexpr int HD_TILE = 256, HD_TOK = DUO_B;
constexpr uint32_t HD_OOB = 0xfffffff0u;   // outside a buffer of any size up to 2^32 - 16 bytes
constexpr float HD_LOG2E = 1.44269504088896340736f, HD_LN2 = 0.69314718055994530942f;
constexpr float HD_FAR = 1024.0f;   // logits from which on their product with log2 e is rounded by 2^-14 or more, up to anything: subtracted before they are multiplied
enum HeadReduction { HD_NONE = 0, HD_MEAN = 1, HD_SUM = 2 };

// ----------------------------------------------------------------------------------------------- the rows that count
struct HeadGather {
    bf16_t *xc;              // [tokens][ldc]: the rows that count, in order, zeros behind their last values; fp32: three planes of ldc / 3 (rdb_duo.hpp)
    const void *x;
    int64_t ldx, ldc;
    const int64_t *target;
    int *pos;                // [tokens]: where a row went, -1: ignored
    const int *counts;       // rows that count of every HD_COUNT, or NULL
    int *count;              // rows that count; behind it the counter of head_merge_kernel's blocks, cleared
    int *label;              // by place: target (-1: none of the classes)
    float *lse, *factor;     // backward, by place, or NULL: logarithm of the row's sum, its own factor of G
    const float *stats;      // lse by row
    const float *dloss;      // [tokens], or NULL: 1
    int64_t tokens, dim, classes, ignore;
    int rows;                // per block
};
__device__ __forceinline__ f32x4 head_load4(const float *p, int left, bool whole)
{
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (whole) __builtin_memcpy(&v, p, 16);   // at any address
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) v[e] = p[e];
    return v;
}
// fg_split3 with products that nobody runs again.  An infinity is (0, 0, infinity): of its six products only that with the other side's first plane is not of zeros, so it is what an
// infinity's is, inf by what is finite and not zero, NaN by zero.  A finite value that would round to an infinity has its first part cut off.  Two comparisons where there is none.
__device__ __forceinline__ void head_split3(float v0, float v1, uint32_t &h, uint32_t &m, uint32_t &l)
{
    constexpr float ROUNDS_UP = 0x1.ffp127f;   // half a step past the largest bf16
    fg_split3(v0, v1, h, m, l);
    if (fabsf(v0) < ROUNDS_UP && fabsf(v1) < ROUNDS_UP) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float v = e ? v1 : v0;
        if (!(fabsf(v) >= ROUNDS_UP)) continue;   // a NaN stays one in the first part
        const int s = 16 * e;
        const uint32_t keep = 0xffffu << (16 - s), bits = __float_as_uint(v);
        uint32_t part[3] = {0u, 0u, bits >> 16};
        if (__builtin_isfinite(v)) {
            part[0] = bits >> 16;
            float r = v - __uint_as_float(bits & 0xffff0000u);
#pragma unroll
            for (int i = 1; i < 3; ++i) {
                part[i] = f32_to_bf16(r);
                r -= __uint_as_float(part[i] << 16);
            }
        }
        h = (h & keep) | part[0] << s;
        m = (m & keep) | part[1] << s;
        l = (l & keep) | part[2] << s;
    }
}
// 8 values, `left` of them there, into the planes
__device__ __forceinline__ void head_split8(bf16_t *to, int plane, const float *from, int left)
{
    const f32x4 a = head_load4(from, left, left >= 4), b = head_load4(from + 4, left - 4, left >= 8);
    u32x4 v[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t h, m, l;
        head_split3(e < 2 ? a[2 * e] : b[2 * e - 4], e < 2 ? a[2 * e + 1] : b[2 * e - 3], h, m, l);
        v[0][e] = h;
        v[1][e] = m;
        v[2][e] = l;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<u32x4 *>(to + i * plane) = v[i];
}
// Blocks count the rows before theirs themselves: 64 KB of targets for the last one of 8192, out of L2.  Of more than HD_COUNTED tokens, where that would grow with their square (2^20: 3700 us
// beside 400 of the logits' launch at 64 -> 1000; 131072: 75; 16384: 16), a launch has counted every HD_COUNT rows (62 and 15 us with it).
constexpr int HD_COUNT = 1024, HD_COUNTED = 16384;
__global__ __launch_bounds__(256) void head_count_kernel(int *__restrict__ counts, const int64_t *__restrict__ target, int64_t tokens, int64_t ignore)
{
    __shared__ int n_[4];
    const int t = threadIdx.x;
    int n = 0;
#pragma unroll
    for (int e = 0; e < HD_COUNT / 256; ++e) {
        const int64_t i = (int64_t)blockIdx.x * HD_COUNT + e * 256 + t;
        n += i < tokens && target[i] != ignore ? 1 : 0;
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) n += __shfl_xor(n, m, 64);
    if ((t & 63) == 0) n_[t >> 6] = n;
    __syncthreads();
    if (t == 0) counts[blockIdx.x] = n_[0] + n_[1] + n_[2] + n_[3];
}
template <bool PLANES> __device__ __forceinline__ void head_gather_rows(const HeadGather &p, int block)
{
    __shared__ int before_[4], place_[64];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t r0 = (int64_t)block * p.rows;
    const int mine = p.tokens - r0 < p.rows ? (int)(p.tokens - r0) : p.rows;
    const int64_t c = wave == 0 && lane < mine ? p.target[r0 + lane] : p.ignore;
    int n = 0;
    int64_t counted = 0;
    if (p.counts) {
        counted = r0 / HD_COUNT * HD_COUNT;
        for (int i = t; i < (int)(r0 / HD_COUNT); i += 256) n += p.counts[i];
    }
#pragma unroll 16
    for (int64_t i = counted + t; i < r0; i += 256) n += p.target[i] != p.ignore ? 1 : 0;
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) n += __shfl_xor(n, m, 64);
    if (lane == 0) before_[wave] = n;
    __syncthreads();
    if (wave == 0) {
        const bool counts = c != p.ignore;
        const unsigned long long all = __ballot(counts);
        const int first = before_[0] + before_[1] + before_[2] + before_[3], at = first + __popcll(all & ((1ull << lane) - 1));
        place_[lane] = counts ? at : -1;
        if (lane < mine) {
            p.pos[r0 + lane] = counts ? at : -1;
            if (counts) {
                const bool known = c >= 0 && c < p.classes;
                p.label[at] = known ? (int)c : -1;
                if (p.lse) {
                    p.lse[at] = p.stats[r0 + lane];
                    p.factor[at] = !known ? __uint_as_float(0x7fc00000u) : p.dloss ? p.dloss[r0 + lane] : 1.0f;
                }
            }
        }
        if (lane == 0 && r0 + mine == p.tokens) {
            p.count[0] = first + __popcll(all);
            p.count[1] = 0;
        }
    }
    __syncthreads();
    if constexpr (PLANES) {
        const int plane = (int)(p.ldc / 3), chunks = plane / 8;
        for (int i = t; i < mine * chunks; i += 256) {
            const int row = i / chunks, col = (i - row * chunks) * 8, at = place_[row];
            if (at >= 0) head_split8(p.xc + (int64_t)at * p.ldc + col, plane, static_cast<const float *>(p.x) + (r0 + row) * p.ldx + col, (int)p.dim - col);
        }
        return;
    }
    const bf16_t *x = static_cast<const bf16_t *>(p.x);
    // 8 values a lane, at any address; a ragged piece of the last row that there is, and rows of less than 8 values, one by one: 16 bytes would reach behind the last of them
    const int chunks = (int)(p.ldc / 8), dim = (int)p.dim, total = mine * chunks, whole = dim < 8 ? 0 : dim % 8 && r0 + mine == p.tokens ? total - 1 : total;
    for (int i0 = t; i0 < whole; i0 += 1024) {
        u32x4 v[4];
        bf16_t *to[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = min(i0 + q * 256, whole - 1), row = i / chunks, col = (i - row * chunks) * 8, at = place_[row], left = dim - col;
            __builtin_memcpy(&v[q], x + (r0 + row) * p.ldx + col, 16);
            to[q] = at < 0 || i0 + q * 256 >= whole ? nullptr : p.xc + (int64_t)at * p.ldc + col;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] &= (2 * e < left ? 0xffffu : 0u) | (2 * e + 1 < left ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (to[q]) *reinterpret_cast<u32x4 *>(to[q]) = v[q];
    }
    for (int i = whole * 8 + t; i < total * 8; i += 256) {
        const int row = i / 8 / chunks, col = i - row * chunks * 8, at = place_[row];
        if (at >= 0) p.xc[(int64_t)at * p.ldc + col] = col < dim ? x[(r0 + row) * p.ldx + col] : (bf16_t)0;
    }
}

// Rows of `cols` bf16 values into rows of a multiple of 8 of them (PAD, zeros behind the last ones) or out of them into rows without gaps; a lane reads 8 values at any address
// and writes them to a multiple of 16 bytes.  per_block: a multiple of 8, of 8192 values or so, or 8 longer rows; out of padded rows it reads up to 14 bytes behind the last of them.
struct HeadRepack {
    bf16_t *dst;
    const void *src;
    int64_t ld, rows;   // of src
    int cols, per_block, blocks;
};
template <bool PAD> __device__ __forceinline__ void head_repack_rows(const HeadRepack &p, int block)
{
    const int64_t r0 = (int64_t)block * p.per_block, lds = p.ld;
    const bf16_t *__restrict__ src = static_cast<const bf16_t *>(p.src);
    bf16_t *__restrict__ dst = p.dst;
    const int cols = p.cols, mine = p.rows - r0 < p.per_block ? (int)(p.rows - r0) : p.per_block, out_cols = PAD ? (cols + 7) & ~7 : cols, total = mine * out_cols;
    src += r0 * lds;
    dst += r0 * out_cols;
    // whole pieces, but for those that would read behind the last row that there is
    const int whole = cols < 8 ? 0 : PAD && r0 + mine == p.rows ? total - out_cols : total & ~7;
    for (int i0 = threadIdx.x * 8; i0 < whole; i0 += 4 * 2048) {
        u32x4 v[4], u[4];
        int left[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = min(i0 + q * 2048, whole - 8), row = i / out_cols, c = i - row * out_cols;
            const bf16_t *from = src + (int64_t)row * lds + c;
            left[q] = cols - c;   // values of this row; the others are zeros, or the next row's first
            __builtin_memcpy(&v[q], from, 16);
            u[q] = u32x4{0u, 0u, 0u, 0u};
            if (!PAD) __builtin_memcpy(&u[q], left[q] < 8 ? from + lds - cols : from, 16);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = i0 + q * 2048;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t m = (2 * e < left[q] ? 0xffffu : 0u) | (2 * e + 1 < left[q] ? 0xffff0000u : 0u);
                v[q][e] = (v[q][e] & m) | (u[q][e] & ~m);
            }
            if (i < whole) *reinterpret_cast<u32x4 *>(dst + i) = v[q];
        }
    }
    for (int i = whole + (int)threadIdx.x; i < total; i += 256) {
        const int row = i / out_cols, c = i - row * out_cols;
        dst[i] = c < cols ? src[(int64_t)row * lds + c] : (bf16_t)0;
    }
}
// The rows that count and, where it needs one, the weight's copy, in one launch (three launches less with dW's, 1025 x 999 -> 10001: a step 136 -> 126.5 us).
// PLANES: fp32, both into planes (50304 x 768: 60 us, 6.4 TB/s).
template <bool PLANES> __global__ __launch_bounds__(256) void head_gather_kernel(HeadGather p, HeadRepack w, int gathering)
{
    if ((int)blockIdx.x < gathering) return head_gather_rows<PLANES>(p, (int)blockIdx.x);
    const int block = (int)blockIdx.x - gathering;
    if constexpr (!PLANES) {
        head_repack_rows<true>(w, block);
    } else {
        const int64_t r0 = (int64_t)block * w.per_block;
        const int mine = w.rows - r0 < w.per_block ? (int)(w.rows - r0) : w.per_block, chunks = (w.cols + 7) / 8;
#pragma unroll 4
        for (int i = threadIdx.x; i < mine * chunks; i += 256) {
            const int row = i / chunks, col = (i - row * chunks) * 8;
            head_split8(w.dst + (r0 + row) * chunks * 24 + col, chunks * 8, static_cast<const float *>(w.src) + (r0 + row) * w.ld + col, w.cols - col);
        }
    }
}

// ----------------------------------------------------------------------------------------------- logits, in the accumulators
struct HeadLogits {
    const bf16_t *x;      // the rows that count, [*count][ldx]
    const bf16_t *w;      // [classes][ldw]
    int64_t ldx, ldw;
    const int *count;     // NULL: all tokens
    unsigned int *cleared;   // NULL, or a word that block 0 sets to zero for a later launch
    int dim, classes, v0;     // classes v0 .. v0 + tiles_v * 256 of this launch
    int tiles_v;
    float2 *part;         // stats: [2 * tiles_v][tokens]: maximum and sum
    float *picked;        // stats, by place: the target's logit, from the tile that has it
    int64_t tokens;
    bf16_t *g;            // gradient: [tokens][ldg], class v0 first
    int64_t ldg;
    int plane, plane_g;   // fp32: values from plane to plane of x and w, of g
    const float *lse, *factor;
    const int *label;
    const int64_t *target;   // few tokens as they are (count NULL): their targets, instead of labels
};
__device__ __forceinline__ int head_row(int j, int g) { return 8 * (j >> 2) + 4 * g + (j & 3); }

// Tiles of MI * 64 classes x NI * 64 tokens, waves 2 x 2.
// Where `ref` is far (classes masked by a type's lowest value, for one), it is taken from v at once: what is returned, or 0 (the other lanes' values keep their bits).
template <int N> __device__ __forceinline__ float head_far(float ref, float (&v)[N])
{
    const float far = fabsf(ref) > HD_FAR ? ref : 0.0f;
    if (__any(far != 0.0f)) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] -= far;
    }
    return far;
}
// Maximum and sum of exponentials relative to it over a wave's `left` classes, of its ni-th 32 tokens.
template <int MI, int NI> __device__ __forceinline__ void head_stats(const f32x16 (&acc)[MI][NI], int ni, int left, int g, float &m, float &s)
{
    constexpr int N = MI * 16;
    float v[N];
    m = -INFINITY;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = acc[i >> 4][ni][i & 15];
    if (left < MI * 32) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((i >> 4) * 32 + head_row(i & 15, g) >= left) v[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float ref = m == -INFINITY ? 0.0f : m, far = head_far(ref, v), scaled = far != 0.0f ? 0.0f : ref * HD_LOG2E;
#pragma unroll
    for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f(fmaf(v[i], HD_LOG2E, -scaled));
    s += __shfl_xor(s, 32, 64);
    s *= __builtin_amdgcn_exp2f(-fmaf(ref - far, HD_LOG2E, -scaled));   // what `scaled` was rounded by
}
__device__ __forceinline__ void head_join(float &m, float &s, float m2, float s2)
{
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top;
    s = s * __builtin_amdgcn_exp2f((m - ref) * HD_LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * HD_LOG2E);
    m = top;
}
// The logit of class `rel` of a wave's, where it has it, of its ni-th 32 tokens.  It has to be the one that is in the sum: from a sum of products in another order nll of a token
// whose own class has nearly all of the probability would be rounding of either sign.
template <int MI, int NI> __device__ __forceinline__ void head_pick(const f32x16 (&acc)[MI][NI], int ni, int rel, int g, float *to)
{
    if (!__any((unsigned)rel < (unsigned)(MI * 32))) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < MI * 16; ++i)
        if ((i >> 4) * 32 + head_row(i & 15, g) == rel) v = acc[i >> 4][ni][i & 15];
    if ((unsigned)rel < (unsigned)(MI * 32) && ((rel >> 2) & 1) == g) *to = v;
}
// A sum has its target's own part, so that what is below zero is rounding.
__device__ __forceinline__ float head_nll(float m, float s, float picked)
{
    const float v = (m - picked) + log2f(s) * HD_LN2;
    return v < 0.0f ? 0.0f : v;
}
__device__ __forceinline__ float head_lse(float m, float s) { return m + log2f(s) * HD_LN2; }
// ... for each of the wave's tokens; each wave leaves its half of the classes' own
template <int MI, int NI>
__device__ __forceinline__ void head_leave_stats(const f32x16 (&acc)[MI][NI], const HeadLogits &p, int tv, int tok0, int count, int t)
{
    const int wave = t >> 6, lane = t & 63, r = lane & 31, g = lane >> 5, wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int tok = tok0 + wn * NI * 32 + ni * 32 + r, first = p.v0 + (tv * 2 + wm) * MI * 32;
        head_pick(acc, ni, tok < count ? p.label[tok] - first : -1, g, p.picked + tok);
        __builtin_amdgcn_sched_barrier(0);
        float m, s;
        head_stats(acc, ni, p.classes - first, g, m, s);
        if (g == 0 && tok < count) p.part[(int64_t)(tv * 2 + wm) * p.tokens + tok] = float2{m, s};
        __builtin_amdgcn_sched_barrier(0);
    }
}

// G of the tile, through LDS into whole rows; classes past the last one are zeros.  PLANES: one plane after the other
template <int MI, int NI, bool PLANES>
__device__ __forceinline__ void head_leave_grad(f32x16 (&acc)[MI][NI], bf16_t *__restrict__ lds, const HeadLogits &p, int tv, int tok0, int count, int t)
{
    constexpr int HALF = MI * 32, N = MI * 16, BM = MI * 64, BN = NI * 64, LD = BM + 8;
    const int wave = t >> 6, lane = t & 63, r = lane & 31, g = lane >> 5, wm = wave >> 1, wn = wave & 1;
    const int first = p.v0 + tv * BM + wm * HALF, left = p.classes - first;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int b = wn * NI * 32 + ni * 32 + r, tok = min(tok0 + b, count - 1);
        const float lse = p.lse[tok], f = p.factor[tok];
        const bool far = fabsf(lse) > HD_FAR;
        const float l = far ? 0.0f : lse * HD_LOG2E;
        if (__any(far)) {   // as head_far; no value above 1, whatever the logits' own rounding, which the forward pass may have had to the other side
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float v = acc[i >> 4][ni][i & 15], d = v - lse;
                acc[i >> 4][ni][i & 15] = !far ? v : d > 0.0f ? 0.0f : d;
            }
        }
        const int rel = p.label[tok] - first;
        if constexpr (PLANES) {   // in place
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i >> 4][ni][i & 15] = __builtin_amdgcn_exp2f(fmaf(acc[i >> 4][ni][i & 15], HD_LOG2E, -l));
            if (__any((unsigned)rel < (unsigned)HALF)) {
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i >> 4][ni][i & 15] -= (i >> 4) * 32 + head_row(i & 15, g) == rel ? 1.0f : 0.0f;
            }
            if (left < HALF) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if ((i >> 4) * 32 + head_row(i & 15, g) >= left) acc[i >> 4][ni][i & 15] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i >> 4][ni][i & 15] *= f;
            __builtin_amdgcn_sched_barrier(0);
            continue;
        }
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_amdgcn_exp2f(fmaf(acc[i >> 4][ni][i & 15], HD_LOG2E, -l));
        if (__any((unsigned)rel < (unsigned)HALF)) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((i >> 4) * 32 + head_row(i & 15, g) == rel) v[i] -= 1.0f;
        }
        if (left < HALF) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((i >> 4) * 32 + head_row(i & 15, g) >= left) v[i] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < MI * 4; ++q)
            store4<bf16_t>(lds + b * LD + wm * HALF + (q >> 2) * 32 + 8 * (q & 3) + 4 * g, v[q * 4] * f, v[q * 4 + 1] * f, v[q * 4 + 2] * f, v[q * 4 + 3] * f);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll 1
    for (int plane = 0; plane < (PLANES ? 3 : 1); ++plane) {
        if constexpr (PLANES) {
            if (plane) __syncthreads();   // the one before is out of LDS
#pragma unroll
            for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                for (int q = 0; q < MI * 4; ++q) {
                    f32x16 &c = acc[q >> 2][ni];
                    const int j = (q & 3) * 4;
                    const uint32_t lo = f32x2_to_bf16x2(c[j], c[j + 1]), hi = f32x2_to_bf16x2(c[j + 2], c[j + 3]);
                    *reinterpret_cast<uint2 *>(lds + (wn * NI * 32 + ni * 32 + r) * LD + wm * HALF + (q >> 2) * 32 + 8 * (q & 3) + 4 * g) = uint2{lo, hi};
                    c[j] -= __uint_as_float(lo << 16);
                    c[j + 1] -= __uint_as_float(lo & 0xffff0000u);
                    c[j + 2] -= __uint_as_float(hi << 16);
                    c[j + 3] -= __uint_as_float(hi & 0xffff0000u);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
        __syncthreads();
        constexpr int LPR = BM / 8, RPP = 256 / LPR;   // lanes a row, rows at once
        bf16_t *out = p.g + (int64_t)tok0 * p.ldg + (int64_t)tv * BM + plane * p.plane_g;
        const int a = (t % LPR) * 8;
#pragma unroll PLANES ? 2 : 8
        for (int q = 0; q < BN / RPP; ++q) {
            const int b = q * RPP + t / LPR;
            if (tok0 + b < count) *reinterpret_cast<f32x4 *>(out + (int64_t)b * p.ldg + a) = *reinterpret_cast<const f32x4 *>(lds + b * LD + a);
        }
    }
}

// Few tokens, one tile of them: bound by the weight, which is read once.  Tiles of 64 classes with four stages of 64 on their way, of 128 with two where these give every
// compute unit a block; statistics by up to two blocks a compute unit, each with several tiles in turn and one part for all of them: parts are what the merging
// kernel's time goes by.  us a forward call, 256 x 64 tiles of rdb_big.hpp | 64 x 64 | 128 x 64 (four stages: 23.5, 32.1, 59.6): 16 tokens x 768 -> 50304 22.7 | 23.8 | 22.3,
// 64 x 4096 -> 16384 57 | 32.1 | 33.1, 32 x 1000 -> 100000 58.6 | 57.0 | 57.2 (77, 134 and 200 MB of weight: 15, 26 and 39 at the rate of a large copy);
// 256 x 128 on two blocks a compute unit 26.1, 75, 60.5.
constexpr int HF_T = 64;
template <bool GRAD, int HF_V> __global__ __launch_bounds__(256, 2) void head_logits_few_kernel(HeadLogits p)
{
    constexpr int MI = HF_V / 64, AHEAD = 4 / MI;
    typedef GlobalOperand<HF_V, 64, K_CONT> PA;
    typedef GlobalOperand<HF_T, 64, K_CONT> PB;
    __shared__ __align__(16) bf16_t lds[2 * (PA::Tile::LDS_ELEMS + PB::Tile::LDS_ELEMS)];
    __shared__ float ms_[2][2][32];
    if (p.cleared && blockIdx.x == 0 && threadIdx.x == 0) *p.cleared = 0u;
    const int count = p.count ? *p.count : (int)p.tokens;
    if (count <= 0) return;
    const int t = threadIdx.x, lane = t & 63, r = lane & 31, g = lane >> 5, wm = t >> 7, wn = (t >> 6) & 1, tok = wn * 32 + r;
    float m = -INFINITY, s = 0.0f;
    int label = -1;
    if (!GRAD && tok < count) {
        const int64_t c = p.target ? p.target[tok] : p.label[tok];
        label = c >= 0 && c < p.classes ? (int)c : -1;
    }
    for (int tv = (int)blockIdx.x; tv < p.tiles_v; tv += (int)gridDim.x) {
        const int row = p.v0 + tv * HF_V, rows = min(HF_V, p.classes - row);
        PA pa = {p.w + (int64_t)row * p.ldw, p.ldw, 0, rows, p.dim, (int64_t)(rows - 1) * p.ldw + p.dim};
        PB pb = {p.x, p.ldx, 0, count, p.dim, (int64_t)(count - 1) * p.ldx + p.dim};
        f32x16 acc[MI][1];
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) acc[mi][0] = zero16();
        gemm_mainloop<HF_V, HF_T, 64, AHEAD, AHEAD>(acc, lds, pa, pb, 0, (p.dim + 63) / 64);
        if constexpr (GRAD) {
            head_leave_grad<MI, 1, false>(acc, lds, p, tv, 0, count, t);
            __syncthreads();
        } else {
            head_pick(acc, 0, label - (row + wm * MI * 32), g, p.picked + tok);
            float m2, s2;
            head_stats(acc, 0, p.classes - (row + wm * MI * 32), g, m2, s2);
            head_join(m, s, m2, s2);
        }
    }
    if constexpr (!GRAD) {
        if (wm == 1 && g == 0) {
            ms_[0][wn][r] = m;
            ms_[1][wn][r] = s;
        }
        __syncthreads();
        if (wm == 0 && g == 0) {
            head_join(m, s, ms_[0][wn][r], ms_[1][wn][r]);
            if (tok < count) p.part[(int64_t)blockIdx.x * p.tokens + tok] = float2{m, s};
        }
    }
}
static int head_few_tile(int64_t classes) { return cdiv(classes, 128) >= num_compute_units() ? 128 : 64; }
static int head_few_blocks(int64_t classes) { return (int)std::min<int64_t>(cdiv(classes, head_few_tile(classes)), 2 * num_compute_units()); }

// The same on two blocks a compute unit, a tile of 256 classes x 128 tokens each.  A die's 64 tiles at a time: 8 of the weight x 8 of the tokens.
template <bool GRAD, bool SOLO, bool PLANES> __device__ __forceinline__ void head_logits_tile(const HeadLogits &p, bf16_t *lds, int count, int block)
{
    const int tiles_t = (count + HD_TOK - 1) / HD_TOK, total = p.tiles_v * tiles_t, per_die = (total + 7) >> 3, w = (block & 7) * per_die + (block >> 3);
    if ((block >> 3) >= per_die || w >= total) return;
    const int per_group = 8 * p.tiles_v, group = w / per_group, in_group = w - group * per_group, size = min(8, tiles_t - group * 8);
    const int tv = in_group / size, tok0 = (group * 8 + in_group - tv * size) * HD_TOK, row = p.v0 + tv * HD_TILE;
    f32x16 acc[DUO_MI][DUO_NI];
    duo_zero(acc);
    const int stages = (p.dim + DUO_K - 1) / DUO_K;
    if constexpr (PLANES) {
        DuoPlanes<DUO_A, K_CONT, 0> pa;
        DuoPlanes<DUO_B, K_CONT, 1> pb;
        pa.set(p.w + (int64_t)row * p.ldw, p.ldw, 0, min(HD_TILE, p.classes - row), p.dim, p.plane);
        pb.set(p.x + (int64_t)tok0 * p.ldx, p.ldx, 0, min(HD_TOK, count - tok0), p.dim, p.plane);
        duo_mainloop<SOLO>(acc, lds, pa, pb, 6 * stages);
    } else {
        DuoOperand<DUO_A, K_CONT> pa;
        DuoOperand<DUO_B, K_CONT> pb;
        pa.set(p.w + (int64_t)row * p.ldw, p.ldw, 0, min(HD_TILE, p.classes - row), p.dim);
        pb.set(p.x + (int64_t)tok0 * p.ldx, p.ldx, 0, min(HD_TOK, count - tok0), p.dim);
        duo_mainloop<SOLO>(acc, lds, pa, pb, stages);
    }
    if constexpr (GRAD) head_leave_grad<DUO_MI, DUO_NI, PLANES>(acc, lds, p, tv, tok0, count, (int)threadIdx.x);
    else head_leave_stats<DUO_MI, DUO_NI>(acc, p, tv, tok0, count, (int)threadIdx.x);
}
// Two blocks a compute unit have 256 registers a lane, accumulators among them: 208 and 222 (head_products_kernel) in bf16; G in planes, whose accumulators are taken apart in place, spills 12 and 13.
template <bool GRAD, bool PLANES> __global__ __launch_bounds__(256, 2) void head_logits_duo_kernel(HeadLogits p)
{
    __shared__ __align__(16) bf16_t lds[DUO_LDS];
    head_logits_tile<GRAD, false, PLANES>(p, lds, p.count ? *p.count : (int)p.tokens, (int)blockIdx.x);
}
template <bool GRAD, bool PLANES> __global__ __launch_bounds__(256, 1) void head_logits_solo_kernel(HeadLogits p)
{
    __shared__ __align__(16) bf16_t lds[SOLO_LDS];
    head_logits_tile<GRAD, true, PLANES>(p, lds, p.count ? *p.count : (int)p.tokens, (int)blockIdx.x);
}

// ----------------------------------------------------------------------------------------------- loss
// What is left of the loss when every row's nll is there: the sum over the rows, in a fixed order, by the block that comes last.  Values pass between blocks on
// different dies, so they are stored and loaded around the dies' caches.
struct HeadSum {
    float *loss;                // one value, or NULL: the rows' own are the loss
    float *count;               // rows that count, as fp32
    float *nll;                 // [tokens]
    unsigned int *arrived;      // 0 when the launch begins
    const int64_t *target;
    int64_t tokens, ignore;
    int mean;
};
__device__ __forceinline__ void head_leave_nll(const HeadSum &p, int64_t row, float v)
{
    if (p.loss) __hip_atomic_store(p.nll + row, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else p.nll[row] = v;
}
// One block of THREADS.
template <int THREADS> __device__ __forceinline__ void head_add_up(const HeadSum &p)
{
    __shared__ float s_[THREADS / 64];
    __shared__ int n_[THREADS / 64];
    const int t = threadIdx.x;
    float a = 0.0f;
    int c = 0;
#pragma unroll 4
    for (int64_t i = t; i < p.tokens; i += THREADS) {
        a += __hip_atomic_load(p.nll + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        c += p.target[i] == p.ignore ? 0 : 1;
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        a += __shfl_xor(a, m, 64);
        c += __shfl_xor(c, m, 64);
    }
    if ((t & 63) == 0) {
        s_[t >> 6] = a;
        n_[t >> 6] = c;
    }
    __syncthreads();
    if (t) return;
    a = 0.0f;
    c = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
        a += s_[w];
        c += n_[w];
    }
    p.loss[0] = p.mean ? a / (float)c : a;
    p.count[0] = (float)c;
}
__global__ __launch_bounds__(1024) void head_loss_kernel(HeadSum p) { head_add_up<1024>(p); }
// The same by the last block of a launch; all THREADS threads of all blocks, after their last head_leave_nll.  Counting one word costs 10 ns a block.
template <int THREADS> __device__ __forceinline__ void head_sum(const HeadSum &p)
{
    __shared__ int last_;
    if (!p.loss) return;
    __builtin_amdgcn_s_waitcnt(0);   // this wave's values are in memory
    __syncthreads();                 // ... and every other wave's
    if (threadIdx.x == 0) last_ = __hip_atomic_fetch_add(p.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (last_) head_add_up<THREADS>(p);
}

struct HeadMerge {
    float *stats;          // [tokens]: lse, 0 in ignored rows
    const float2 *part;    // [parts][tokens], by place
    const float *picked;   // by place
    const int *pos;        // NULL: every row in its place
    int64_t classes;
    int parts;
    HeadSum sum;
};
// LANES lanes a token: many where the tokens are few and their parts a chain of loads.
template <int LANES> __global__ __launch_bounds__(1024) void head_merge_kernel(HeadMerge p)
{
    constexpr int TOK = 1024 / LANES;
    __shared__ float ms_[TOK][LANES + 1], ss_[TOK][LANES + 1];
    const int t = threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.x * TOK, tokens = p.sum.tokens;
    auto place = [&](int64_t row) { return row >= tokens ? -1 : p.pos ? p.pos[row] : p.sum.target[row] == p.sum.ignore ? -1 : (int)row; };
    {   // neighbouring lanes: neighbouring tokens, as the parts lie; then over to the token's own lanes
        const int tok = t % TOK, slot = t / TOK, at = place(r0 + tok);
        float m = -INFINITY, s = 0.0f;
        if (at >= 0)
#pragma unroll 8
            for (int i = slot; i < p.parts; i += LANES) {
                const float2 q = p.part[(int64_t)i * tokens + at];
                head_join(m, s, q.x, q.y);
            }
        ms_[tok][slot] = m;
        ss_[tok][slot] = s;
    }
    __syncthreads();
    const int tok = t / LANES, lane = t % LANES, at = place(r0 + tok);
    const int64_t row = r0 + tok;
    float m = ms_[tok][lane], s = ss_[tok][lane];
    const int64_t c = at < 0 ? 0 : p.sum.target[row];
    const bool known = c >= 0 && c < p.classes;
    const float picked = at >= 0 && known && lane == 0 ? p.picked[at] : 0.0f;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) head_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    if (lane == 0 && row < tokens) {
        p.stats[row] = at < 0 ? 0.0f : head_lse(m, s);
        head_leave_nll(p.sum, row, at < 0 ? 0.0f : known ? head_nll(m, s, picked) : __uint_as_float(0x7fc00000u));
    }
    head_sum<1024>(p.sum);
}

// ----------------------------------------------------------------------------------------------- dx and dW
// The factor that all of G's rows share.  No rows: nothing to scale.
struct HeadScale {
    const float *dloss;   // NULL: 1 (rows have factors of their own)
    const float *count;   // NULL: a sum
    __device__ __forceinline__ float value() const { return !dloss ? 1.0f : !count ? dloss[0] : count[0] > 0.0f ? dloss[0] / count[0] : 0.0f; }
};
struct HeadProducts {
    const bf16_t *g, *x, *w;   // w: the piece's first class
    int64_t ldg, ldx, ldw;
    const int *count;
    int rows_v, dim;           // classes of the piece
    float *dx;                 // [splits][tokens][lddx] sums, or NULL
    int64_t lddx, dx_stride, tokens;
    bool add;                  // to the sums that are there
    int splits, split_v;       // a split's classes, a multiple of 64
    void *dw;                  // the piece's first row of [classes][lddw], or NULL
    int plane, plane_g;        // fp32: as in HeadLogits
    int64_t lddw;
    HeadScale scale;
    int tiles_d, tiles_v;
    int blocks_dw, blocks_dx;   // of the launch, multiples of 8; the others are the next piece's logits
};
// D[a][b] to out[a * ld + b], times a factor (KEEP: fp32 sums, which the next launch adds to or finds, as they are; ADD: added to what is there): each wave passes 32 rows x
// its 64 columns at a time through LDS, so that a lane stores 16 bytes of a row
template <typename E, bool KEEP, bool ADD>
__device__ __forceinline__ void head_store_rows(f32x16 (&acc)[DUO_MI][DUO_NI], bf16_t *__restrict__ lds, E *__restrict__ out, int64_t ld, int na, int b0, int nb, float scale, int t)
{
    constexpr int COLS = DUO_NI * 32, LDP = COLS + 4, PER = 16 / (int)sizeof(E), LPR = COLS / PER, RPP = 64 / LPR;
    const int wave = t >> 6, lane = t & 63, r = lane & 31, g = lane >> 5, wm = wave >> 1, wn = wave & 1;
    float *patch = reinterpret_cast<float *>(lds) + wave * 32 * LDP;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(out, 0, (int)(((int64_t)(na - 1) * ld + nb) * (int)sizeof(E)), 0x00020000);
    const int col = (lane % LPR) * PER, b = b0 + wn * COLS + col;
#pragma unroll
    for (int mi = 0; mi < DUO_MI; ++mi) {
#pragma unroll
        for (int ni = 0; ni < DUO_NI; ++ni)
#pragma unroll
            for (int j = 0; j < 16; ++j) patch[head_row(j, g) * LDP + ni * 32 + r] = acc[mi][ni][j];
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_wave_barrier();   // LDS serves a wave's instructions in order: the reads see these writes
#pragma unroll
        for (int q = 0; q < 32 / RPP; ++q) {
            const int row = q * RPP + lane / LPR, a = wm * DUO_MI * 32 + mi * 32 + row;
            const uint32_t off = (a < na && b < nb) ? (uint32_t)(((int64_t)a * ld + b) * (int)sizeof(E)) : HD_OOB;
            f32x4 v = *reinterpret_cast<const f32x4 *>(patch + row * LDP + col);
            if constexpr (sizeof(E) == 2) {
                const f32x4 u = *reinterpret_cast<const f32x4 *>(patch + row * LDP + col + 4);
                const i32x4 h = {(int)f32x2_to_bf16x2(v[0] * scale, v[1] * scale), (int)f32x2_to_bf16x2(v[2] * scale, v[3] * scale),
                                 (int)f32x2_to_bf16x2(u[0] * scale, u[1] * scale), (int)f32x2_to_bf16x2(u[2] * scale, u[3] * scale)};
                __builtin_amdgcn_raw_buffer_store_b128(h, rs, (int)off, 0, 2);
            } else {
                if (ADD) {
                    const f32x4 o = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += o[e];
                }
                if constexpr (KEEP) {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, v), rs, (int)off, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] *= scale;
                    if (b + 4 <= nb) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, v), rs, (int)off, 0, 2);
                    else   // the last values of a row
#pragma unroll
                        for (int e = 0; e < 3; ++e) __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(v[e]), rs, a < na && b + e < nb ? (int)(off + 4u * e) : (int)HD_OOB, 0, 0);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// dW's tiles (256 classes x 128 columns), dx's (256 tokens x 128 columns, a range of the piece's classes), and the next piece's logits: short tiles that fill the
// compute units that have no more of the long ones.
template <bool ADD, bool PLANES> __global__ __launch_bounds__(256, 2) void head_products_kernel(HeadProducts p, HeadLogits next)
{
    __shared__ __align__(16) bf16_t lds[DUO_LDS];
    const int count = *p.count;
    int block = (int)blockIdx.x;
    if (block >= p.blocks_dw + p.blocks_dx) return head_logits_tile<true, false, PLANES>(next, lds, count, block - p.blocks_dw - p.blocks_dx);
    const bool dw = block < p.blocks_dw;
    if (!dw) block -= p.blocks_dw;
    const int tiles_t = (count + HD_TILE - 1) / HD_TILE, n = (dw ? p.tiles_v : p.splits * tiles_t) * p.tiles_d, per_die = (n + 7) >> 3, w = (block & 7) * per_die + (block >> 3);
    if ((block >> 3) >= per_die || w >= n) return;
    f32x16 acc[DUO_MI][DUO_NI];
    duo_zero(acc);
    const int td = w % p.tiles_d, b0 = td * DUO_B;
    if (dw) {
        const int tv = w / p.tiles_d;
        const int stages = (count + DUO_K - 1) / DUO_K, rows = min(HD_TILE, p.rows_v - tv * HD_TILE);   // no rows: zeros
        if constexpr (PLANES) {
            DuoPlanes<DUO_A, M_CONT, 0> pa;   // G: rows = classes, contraction = tokens
            DuoPlanes<DUO_B, M_CONT, 1> pb;   // x: rows = its columns
            pa.set(p.g, p.ldg, tv * HD_TILE, (int)p.ldg, count, p.plane_g);
            pb.set(p.x, p.ldx, b0, (int)p.ldx, count, p.plane);
            duo_mainloop<false>(acc, lds, pa, pb, 6 * stages);
            head_store_rows<float, false, false>(acc, lds, static_cast<float *>(p.dw) + (int64_t)tv * HD_TILE * p.lddw, p.lddw, rows, b0, (int)p.lddw, p.scale.value(), (int)threadIdx.x);
        } else {
            DuoOperand<DUO_A, M_CONT> pa;
            DuoOperand<DUO_B, M_CONT> pb;
            pa.set(p.g, p.ldg, tv * HD_TILE, (int)p.ldg, count);
            pb.set(p.x, p.ldx, b0, p.dim, count);
            duo_mainloop<false>(acc, lds, pa, pb, stages);
            head_store_rows<bf16_t, false, false>(acc, lds, static_cast<bf16_t *>(p.dw) + (int64_t)tv * HD_TILE * p.lddw, p.lddw, rows, b0, p.dim, p.scale.value(), (int)threadIdx.x);
        }
    } else {
        const int tt = w / p.tiles_d % tiles_t, s = w / p.tiles_d / tiles_t, v0 = s * p.split_v, vs = min(p.split_v, p.rows_v - v0), tok = tt * HD_TILE;
        const int toks = min(HD_TILE, count - tok), stages = (vs + DUO_K - 1) / DUO_K;
        if constexpr (PLANES) {
            DuoPlanes<DUO_A, K_CONT, 0> pa;   // G: rows = tokens, contraction = classes
            DuoPlanes<DUO_B, M_CONT, 1> pb;   // W: rows = its columns
            pa.set(p.g + (int64_t)tok * p.ldg + v0, p.ldg, 0, toks, (vs + 7) & ~7, p.plane_g);
            pb.set(p.w + (int64_t)v0 * p.ldw, p.ldw, b0, (int)p.ldw, vs, p.plane);
            duo_mainloop<false>(acc, lds, pa, pb, 6 * stages);
        } else {
            DuoOperand<DUO_A, K_CONT> pa;
            DuoOperand<DUO_B, M_CONT> pb;
            pa.set(p.g + (int64_t)tok * p.ldg + v0, p.ldg, 0, toks, (vs + 7) & ~7);
            pb.set(p.w + (int64_t)v0 * p.ldw, p.ldw, b0, p.dim, vs);
            duo_mainloop<false>(acc, lds, pa, pb, stages);
        }
        head_store_rows<float, true, ADD>(acc, lds, p.dx + s * p.dx_stride + (int64_t)tok * p.lddx, p.lddx, toks, b0, p.dim, 1.0f, (int)threadIdx.x);
    }
}

// dx[row] = factor * the sums of its place over the splits, rounded once; zeros in ignored rows.  The blocks behind those bring dW into rows without gaps.
template <typename E> __global__ __launch_bounds__(256) void head_dx_kernel(E *__restrict__ dx, const float *__restrict__ sums, const int *__restrict__ pos, int64_t tokens, int dim,
                                                      int64_t ld, int64_t stride, int splits, HeadScale scale, HeadRepack dw)
{
    const int summing = (int)gridDim.x - dw.blocks;
    if ((int)blockIdx.x >= summing) return head_repack_rows<false>(dw, (int)blockIdx.x - summing);
    const float f = scale.value();
    const int chunks = (int)(ld / 4);
    const int64_t n = tokens * chunks;
    const bool whole = dim % 4 == 0;   // rows of dx begin on pieces of 4 values then
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)summing * 256) {
        const int64_t row = i / chunks;
        const int c = (int)(i - row * chunks) * 4, at = pos[row];
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (at >= 0) {
#pragma unroll 8
            for (int s = 0; s < splits; ++s) {
                const f32x4 u = *reinterpret_cast<const f32x4 *>(sums + s * stride + at * ld + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += u[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= f;
        }
        E *out = dx + row * dim + c;
        if (whole) {
            if (c >= dim) continue;
            if constexpr (sizeof(E) == 4) *reinterpret_cast<f32x4 *>(out) = v;
            else *reinterpret_cast<uint2 *>(out) = uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < dim) {
                    if constexpr (sizeof(E) == 4) out[e] = v[e];
                    else out[e] = f32_to_bf16(v[e]);
                }
        }
    }
}

// ----------------------------------------------------------------------------------------------- fp32: rows of a piece of logits
struct HeadRows {
    float *logits;         // [tokens][n], n classes from v0 on
    float *g;              // G, there or somewhere else
    float2 *state;         // [tokens]: maximum and sum of the pieces so far
    float *picked;         // [tokens]: the target's logit
    float *stats;
    int64_t classes;
    int n, v0, first, last, columns;
    HeadSum sum;           // tokens and targets; the last piece: nll
    // gradient
    HeadScale scale;
    const float *dloss;    // [tokens], or NULL
    float *xc;             // NULL, or where a row of x goes, zeros for an ignored one
    const float *x;
    int64_t ldx;
    int dim;
};
// One block a row.
template <int THREADS> __global__ __launch_bounds__(THREADS) void head_rows_stats_kernel(HeadRows p)
{
    __shared__ float ms_[THREADS / 64], ss_[THREADS / 64];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x;
    const int64_t c = p.sum.target[row];
    const bool counts = c != p.sum.ignore, known = c >= 0 && c < p.classes;
    const float *l = p.logits + row * p.n;
    float m = -INFINITY, s = 0.0f;
    if (counts)
#pragma unroll 4
        for (int i = t; i < p.n; i += THREADS) {
            const float v = l[i], top = fmaxf(m, v), ref = top == -INFINITY ? 0.0f : top;
            s = s * __expf(m - ref) + __expf(v - ref);
            m = top;
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) head_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    if ((t & 63) == 0) {
        ms_[t >> 6] = m;
        ss_[t >> 6] = s;
    }
    __syncthreads();
    if (t) return;
    for (int w = 1; w < THREADS / 64; ++w) head_join(m, s, ms_[w], ss_[w]);
    if (!p.first && counts) head_join(m, s, p.state[row].x, p.state[row].y);
    float picked = p.first || !known || !counts ? 0.0f : p.picked[row];
    if (counts && known && c >= p.v0 && c < p.v0 + p.n) picked = l[c - p.v0];
    if (p.last) {
        p.stats[row] = counts ? head_lse(m, s) : 0.0f;
        head_leave_nll(p.sum, row, !counts ? 0.0f : known ? head_nll(m, s, picked) : __uint_as_float(0x7fc00000u));
    } else {
        p.state[row] = float2{m, s};
        p.picked[row] = picked;
    }
}
// p.columns of a row a block
__global__ __launch_bounds__(256) void head_rows_grad_kernel(HeadRows p)
{
    const int64_t row = blockIdx.x, c = p.sum.target[row];
    const bool counts = c != p.sum.ignore, known = c >= 0 && c < p.classes;
    const float *l = p.logits + row * p.n;
    float *out = p.g + row * p.n;
    const float lse = p.stats[row], f = !counts ? 0.0f : !known ? __uint_as_float(0x7fc00000u) : p.dloss ? p.dloss[row] : p.scale.value();
    const int label = known ? (int)(c - p.v0) : -1, begin = (int)blockIdx.y * p.columns, end = min(p.n, begin + p.columns);
    if (counts)
#pragma unroll 4
        for (int i = begin + (int)threadIdx.x; i < end; i += 256) {
            const float e = expf(l[i] - lse);
            float v = e > 1.0f ? 1.0f : e;   // logits of another kernel's may be rounded to the other side
            if (i == label) v -= 1.0f;
            out[i] = v * f;
        }
    else
        for (int i = begin + (int)threadIdx.x; i < end; i += 256) out[i] = 0.0f;
    if (p.xc && blockIdx.y == 0)
        for (int i = threadIdx.x; i < p.dim; i += 256) p.xc[row * p.dim + i] = counts ? p.x[row * p.ldx + i] : 0.0f;
}
__global__ __launch_bounds__(256) void head_add_kernel(float *__restrict__ out, const float *__restrict__ a, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] += a[i];
}

// fp32, up to 32 tokens: both products that read the weight, bound by reading it, on the fp32 matrix instructions, which here are faster than splitting the weight for the bf16 ones.
// us a product, split | these: 12 tokens x 2048 -> 47643 (390 MB, 70 by reading alone) logits 144 | 100, dx 142 | 95; steps of 3 x 1024 -> 72064 389 | 350, 32 x 1024 -> 30000
// 167 | 163.  With two tiles of tokens they lose (64 x 1024 -> 30000: logits 44 | 87); without the way through LDS, each lane reading a row, the logits take 142.
constexpr int HS_T = 32;   // tokens, at most
struct HeadFew {
    const float *x, *w;    // logits: hidden states [tokens][ldx]; dx: G
    int64_t ldx, ldw;
    float *out;            // logits [tokens][classes]; dx: [ranges][tokens][dim] sums
    int tokens, dim, classes;
    int range;             // dx: classes of a range, a multiple of 32
};
// The waves' sums one after the other: deterministic.  COLS values a token.
template <int COLS, typename F> __device__ __forceinline__ void head_add_waves(float (&sums)[HS_T][COLS + 4], int wave, F value)
{
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (wave == w) value([&](int tok, int col, float v) { sums[tok][col] = w ? sums[tok][col] + v : v; });
        __syncthreads();
    }
}
// Logits of 64 classes: a wave takes every fourth 32 of the contraction, in whole lines of memory, through LDS of its own (16-byte piece c of row r at c ^ (r & 7)); a lane has four
// neighbours of a class's row and of a token's there (which instruction multiplies which of them is the same for both).
__global__ __launch_bounds__(256, 2) void head_few_logits_kernel(HeadFew p)
{
    constexpr int V = 64, ROWS = V + HS_T, LOADS = ROWS / 8;
    __shared__ __align__(16) float rows_[4][ROWS * 32];
    __shared__ float sums[HS_T][V + 4];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, r = lane & 31, g = lane >> 5, v0 = (int)blockIdx.x * V, piece = lane & 7;
    const float *from[LOADS];
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
        const int row = q * 8 + (lane >> 3);
        from[q] = row < V ? p.w + (int64_t)min(v0 + row, p.classes - 1) * p.ldw : p.x + (int64_t)min(row - V, p.tokens - 1) * p.ldx;
    }
    float *lds = rows_[wave], *to = lds + (lane >> 3) * 32 + (piece ^ (lane >> 3)) * 4;
    f32x16 acc[2] = {zero16(), zero16()};
    f32x4 next[LOADS];
    auto load = [&](int k) {
        const bool whole = k + 32 <= p.dim;
        const int at = k + piece * 4;
#pragma unroll
        for (int q = 0; q < LOADS; ++q) next[q] = head_load4(from[q] + at, p.dim - at, whole);
    };
    load(wave * 32);
    for (int k = wave * 32; k < p.dim; k += 128) {   // behind the last value: zeros
#pragma unroll
        for (int q = 0; q < LOADS; ++q) *reinterpret_cast<f32x4 *>(to + q * 256) = next[q];
        load(k + 128);
        __builtin_amdgcn_wave_barrier();   // LDS serves a wave's instructions in order: the reads see these writes, and the next writes come behind the reads
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 v[3];
#pragma unroll
            for (int m = 0; m < 3; ++m) v[m] = *reinterpret_cast<const f32x4 *>(lds + (m * 32 + r) * 32 + (((q * 2 + g) ^ (r & 7)) * 4));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int mi = 0; mi < 2; ++mi) acc[mi] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[mi][e], v[2][e], acc[mi], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
    }
    head_add_waves<V>(sums, wave, [&](auto add) {
#pragma unroll
        for (int mi = 0; mi < 2; ++mi)
#pragma unroll
            for (int j = 0; j < 16; ++j) add(r, mi * 32 + head_row(j, g), acc[mi][j]);
    });
    for (int i = t; i < HS_T * V; i += 256) {
        const int tok = i / V, v = i % V;
        if (tok < p.tokens && v0 + v < p.classes) p.out[(int64_t)tok * p.classes + v0 + v] = sums[tok][v];
    }
}
// dx, 128 columns and a range of the classes: a wave takes every fourth 8 of them, a lane four neighbouring columns of a class's row, which go to four accumulators.
__global__ __launch_bounds__(256, 2) void head_few_dx_kernel(HeadFew p)
{
    __shared__ float sums[HS_T][128 + 4];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, r = lane & 31, g = lane >> 5, d0 = (int)blockIdx.x * 128, d = d0 + r * 4;
    const int begin = (int)blockIdx.y * p.range, end = min(p.classes, begin + p.range), left = p.dim - d;
    const float *w = p.w + d, *x = p.x + (int64_t)min(r, p.tokens - 1) * p.ldx;   // columns behind the last are not read
    f32x16 acc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = zero16();
    f32x4 a[2][4], b[2];
    auto load = [&](int i, int v) {
        const bool whole = v + 8 <= end, columns = whole && left >= 4;
        v += g * 4;
#pragma unroll
        for (int s = 0; s < 4; ++s) a[i][s] = head_load4(w + (int64_t)min(v + s, p.classes - 1) * p.ldw, v + s < end ? left : 0, columns);
        b[i] = head_load4(x + v, end - v, whole);
    };
    auto multiply = [&](int i) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i][s][e], b[i][s], acc[e], 0, 0, 0);
    };
    load(0, begin + wave * 8);
    for (int v = begin + wave * 8; v < end; v += 64) {
        load(1, v + 32);
        multiply(0);
        load(0, v + 64);
        multiply(1);
    }
    head_add_waves<128>(sums, wave, [&](auto add) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 16; ++j) add(r, 4 * head_row(j, g) + e, acc[e][j]);
    });
    float *out = p.out + (int64_t)blockIdx.y * p.tokens * p.dim;
    for (int i = t; i < HS_T * 128; i += 256) {
        const int tok = i / 128, c = d0 + i % 128;
        if (tok < p.tokens && c < p.dim) out[(int64_t)tok * p.dim + c] = sums[tok][i % 128];
    }
}
// out = the ranges' sums, and what is there
__global__ __launch_bounds__(256) void head_few_sum_kernel(float *__restrict__ out, const float *__restrict__ sums, int64_t n, int ranges, bool add)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = add ? out[i] : 0.0f;
#pragma unroll 8
    for (int s = 0; s < ranges; ++s) v += sums[s * n + i];
    out[i] = v;
}

// ----------------------------------------------------------------------------------------------- plan and calls
// Bytes of a piece's G (bf16) or logits (fp32).  Such an amount the next launch finds in the chip's last-level cache.  A piece of G is twice or four times as large where
// its launch (dW, dx and the next piece's logits) would otherwise end with dW's tiles, which contract all tokens: in units of a stage of 64, as long as a block
// has, on average, less than twice the length of one.  8192 tokens -> 50304, us a step with pieces of 128, 256, 384, 512, 1024 MB: 256 columns 1472, 1222, 1118, 1034, 1097;
// 768 columns 2319, 2319, 2329, 2322, 2449; 4096 tokens x 4096 -> 65536 7076, 7082, 7090, 7138, 7134.
constexpr int64_t HD_PIECE_BYTES = 128ll << 20, HD_PIECE_MOST = 512ll << 20;
constexpr int HD_TILE_COST = 8;   // of a tile's first operands and its stores
// planes: 1, or 3 of fp32, with six products of them
static int64_t head_piece_bytes(int64_t tokens, int64_t dim, int64_t planes)
{
    const int64_t products = planes == 1 ? 1 : 6, td = cdiv(dim, DUO_B), longest = products * cdiv(tokens, DUO_K) + HD_TILE_COST;
    const int64_t of_256 = td * longest + cdiv(tokens, HD_TILE) * td * products * (HD_TILE / DUO_K) + cdiv(tokens, HD_TOK) * (products * cdiv(dim, DUO_K) + HD_TILE_COST);   // work of 256 classes
    int64_t bytes = HD_PIECE_BYTES;
    while (bytes < HD_PIECE_MOST && bytes / (2 * planes * HD_TILE * tokens) * of_256 < 2 * longest * 2 * num_compute_units()) bytes *= 2;
    return bytes;
}

// The logits of few tokens beside the weight are kept for the backward call.
static bool head_keepable(int64_t tokens, int64_t dim, int64_t classes) { return 4 * tokens <= dim && tokens * classes <= (1ll << 26); }
// fp32 on the tiles of the bf16 products, x, W and G in three planes each and six products of them, 1.1 - 1.25 PFLOP/s of bf16, where the offsets allow it and there are tiles enough:
// in the logits two a compute unit, in dW (which contracts all tokens) three to four units in a piece, of not so few tokens that most of a tile of dx is for none.  Otherwise the
// products of rdb_f32.hip, with smaller tiles and long contractions in ranges.  us, those | planes, forward: 2048 x 768 -> 50304 915 | 808, 8192 x 768 -> 50304 3554 | 2906, 3135 x 64 -> 5696
// 44 | 29, 1000 x 512 -> 8000 64 | 62, 1024 x 2048 -> 8000 193 | 205, 2000 x 256 -> 2000 32 | 38; a step: 2048 x 768 -> 50304 3730 | 3420, 8192 x 768 -> 50304 16240 | 13380, 768 x 512 ->
// 20000 491 | 412, 700 x 768 -> 30000 876 | 893, 400 x 512 -> 60000 769 | 917, 1024 x 1024 -> 4000 237 | 295, 8192 x 128 -> 30000 2382 | 3893.  Rows that are ignored cost nothing in planes:
// 645 x 320 -> 103808 with half of them 1489 | 991.  Not where fp32 matrix instructions are asked for (rdb_set_f32_split).
static bool head_in_planes(int64_t tokens, int64_t dim, int64_t classes, bool backward)
{
    const int64_t row = 3 * (dim + 7);
    if (!f32_split_mode() || tokens <= HS_T || tokens > (1ll << 20) || head_keepable(tokens, dim, classes) || row >= (1ll << 20) || row * std::max<int64_t>(tokens, HD_TILE) >= (1ll << 29)) return false;
    const int64_t units = num_compute_units();
    if (!backward) return cdiv(classes, HD_TILE) * cdiv(tokens, HD_TOK) >= 2 * units;
    return tokens >= 576 && std::min(classes, HD_PIECE_MOST / (6 * tokens)) / HD_TILE * cdiv(dim, DUO_B) >= units / 4 * 3;
}

struct HeadPlan {
    int64_t tokens, dim, classes;
    int dtype;
    bool backward, want_dx, want_dw, pack_w, pad_dw;
    bool direct;               // few tokens, forward: x as it is, ignored rows and all
    bool tiles;                // on the tiles of rdb_duo.hpp (few: rdb_gemm.hpp)
    int64_t planes;            // of an operand there: 1, or 3 (fp32)
    int64_t dp, vp;            // columns of the copies; classes of a piece
    int pieces, splits;
    bool few;                  // one tile of few tokens
    int64_t range;             // fp32, few: classes of a range of dx
    int parts;                 // of a token's sum
    int64_t split_v;
    // offsets in the workspace
    int64_t xc, pos, counts, count, lse, factor, label, wc, part, nll, picked, g, dx, dw, product, product_bytes, total;
};
// Tokens up to which a copy of the rows that count costs more than leaving some out gains: one tile of tokens either way.
constexpr int64_t HD_FEW = HF_T;

static HeadPlan head_plan(int64_t tokens, int64_t dim, int64_t classes, int dtype, int64_t ldw, bool backward, bool want_dx, bool want_dw, bool wide_x, bool pack_w, bool kept)
{
    HeadPlan h = {};
    h.tokens = tokens;
    h.dim = dim;
    h.classes = classes;
    h.dtype = dtype;
    h.backward = backward;
    h.want_dx = want_dx;
    h.want_dw = want_dw;
    h.planes = dtype == RDB_F32 && head_in_planes(tokens, dim, classes, backward) ? 3 : 1;
    h.tiles = dtype != RDB_F32 || h.planes > 1;
    const bool f32 = !h.tiles;
    h.dp = f32 ? dim : (dim + 7) / 8 * 8;
    h.pack_w = h.tiles && (pack_w || h.planes > 1);
    h.pad_dw = dtype != RDB_F32 && h.dp != dim;
    const int64_t es = f32 ? 4 : 2 * h.planes;   // bytes of a value of G
    int64_t cols = (f32 ? 2 * HD_PIECE_BYTES : head_piece_bytes(tokens, dim, h.planes)) / (es * tokens) / HD_TILE * HD_TILE;
    // 32-bit offsets within a piece of the weight, of dW, and of G with 128 tokens more
    const int64_t far = h.pack_w ? h.planes * h.dp : std::max(h.dp, ldw);
    cols = std::min<int64_t>(cols, (f32 ? (1ll << 29) - 1 : 1ll << 28) / std::max(f32 ? tokens : 0, far) / HD_TILE * HD_TILE);
    if (h.tiles) cols = std::min<int64_t>(cols, (1ll << 23) / h.planes / HD_TILE * HD_TILE);
    cols = std::max<int64_t>(cols, HD_TILE);
    h.pieces = (int)cdiv(classes, cols);
    h.vp = cdiv(cdiv(classes, h.pieces), HD_TILE) * HD_TILE;
    if (f32 && h.pieces == 1) h.vp = classes;
    h.pieces = (int)cdiv(classes, h.vp);
    h.few = tokens <= HD_FEW && h.planes == 1;
    if (f32 && tokens <= HS_T) {   // ranges of dx: four blocks a compute unit, at least 128 classes each, sums of at most an eighth of the weight's bytes
        const int64_t most = std::min(4 * num_compute_units() / cdiv(dim, 128), std::min(h.vp / 128, h.vp / (8 * tokens)));
        h.range = cdiv(cdiv(h.vp, std::max<int64_t>(1, most)), 32) * 32;
    }
    const int64_t tiles = cdiv(tokens, HD_TILE) * cdiv(dim, DUO_B);
    // Ranges of the classes, each with sums of dx of its own, until every block slot has a tile: at least 4 stages each, and 16 ranges or 16 MB of sums (24 tokens x 960 ->
    // 39040: 16 ranges of 38 stages 60 us, 64 of 10 35; 5 x 64 -> 1792: one of 28 24 us, 7 of 4 7).
    int64_t splits = std::max<int64_t>(1, 2 * num_compute_units() / std::max<int64_t>(1, tiles));
    splits = std::min(splits, cdiv(std::min(h.vp, classes), 4 * DUO_K));
    splits = std::min(splits, std::max<int64_t>(16, std::min<int64_t>(64, (16ll << 20) / (tokens * h.dp * 4))));
    h.split_v = cdiv(cdiv(h.vp, splits), 64) * 64;
    h.splits = (int)cdiv(std::min(h.vp, classes), h.split_v);   // the first piece's: it writes all the sums that there are
    int64_t at = 0;
    auto room = [&](int64_t bytes) {
        const int64_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    };
    h.direct = dtype != RDB_F32 && !backward && tokens <= HD_FEW && wide_x;
    if (f32 ? want_dw : !h.direct) h.xc = room(tokens * h.dp * es);
    if (!f32 && !h.direct) h.pos = room(tokens * 4);
    if (!f32 && tokens > HD_COUNTED) h.counts = room(cdiv(tokens, HD_COUNT) * 4);
    h.count = room(8);
    if (h.pack_w) h.wc = room(classes * h.dp * 2 * h.planes);
    if (!backward) {
        h.nll = room(tokens * 4);
        if (f32) {
            h.part = room(tokens * 8);
            h.picked = room(tokens * 4);
            if (!kept) h.g = room(tokens * h.vp * 4);   // logits that are kept have a buffer of the caller's
        } else {
            if (!h.direct) h.label = room(tokens * 4);
            h.picked = room(tokens * 4);
            h.parts = h.few ? head_few_blocks(classes) : (int)(2 * cdiv(classes, HD_TILE));
            h.part = room(h.parts * tokens * 8);
        }
    } else {
        if (!f32) {
            h.lse = room(tokens * 4);
            h.factor = room(tokens * 4);
            h.label = room(tokens * 4);
        }
        h.g = room(tokens * h.vp * es * (!f32 && h.pieces > 1 ? 2 : 1));   // bf16: a piece's, and the next one's beside it
        if (want_dx && (!f32 || h.range || h.pieces > 1)) h.dx = room((!f32 ? h.splits : h.range ? cdiv(h.vp, h.range) : 1) * tokens * h.dp * 4);
        if (want_dw && h.pad_dw) h.dw = room(classes * h.dp * 2 + 16);
    }
    if (f32) {
        h.product_bytes = rdb_product_f32_workspace_bytes(tokens, h.vp, dim);
        if (h.pieces > 1) h.product_bytes = std::max(h.product_bytes, rdb_product_f32_workspace_bytes(tokens, classes - (h.pieces - 1) * h.vp, dim));
        if (backward)
            for (int64_t n : {h.vp, classes - (h.pieces - 1) * h.vp}) {
                if (want_dx) h.product_bytes = std::max(h.product_bytes, rdb_product_f32_workspace_bytes(tokens, dim, n));
                if (want_dw) h.product_bytes = std::max(h.product_bytes, rdb_product_f32_workspace_bytes(n, dim, tokens));
            }
        h.product = room(h.product_bytes);
    }
    h.total = at;
    return h;
}

struct HeadCall {
    const HeadPlan &h;
    char *ws;
    const void *x, *w;
    int64_t ldx, ldw;
    const int64_t *target;
    int64_t ignore;
    hipStream_t s;
    template <typename T> T *at(int64_t offset) const { return reinterpret_cast<T *>(ws + offset); }
};
static bool head_aligned(const void *p, int64_t ld, int es) { return !((uintptr_t)p & 15) && ld * es % 16 == 0; }

static HeadRepack head_repack(bf16_t *dst, const void *src, int64_t ld, int64_t rows, int64_t cols)
{
    const int64_t per_block = std::max<int64_t>(1, 1024 / cols) * 8;   // four pieces a lane
    return {dst, src, ld, rows, (int)cols, (int)per_block, (int)cdiv(rows, per_block)};
}
// The rows that count and the weight as the tiles read it: rows from 16-byte boundaries on
static int head_gather(const HeadCall &c, const float *stats, const float *dloss_rows, const bf16_t **w, int64_t *ldw)
{
    const HeadPlan &h = c.h;
    HeadGather p = {};
    HeadRepack r = {};
    int64_t gathering = 0;
    *w = static_cast<const bf16_t *>(c.w);
    *ldw = c.ldw;
    if (h.pack_w) {
        r = head_repack(c.at<bf16_t>(h.wc), c.w, c.ldw, h.classes, h.dim);
        *w = r.dst;
        *ldw = h.planes * h.dp;
    }
    if (!h.direct) {
        p.xc = c.at<bf16_t>(h.xc);
        p.x = c.x;
        p.ldx = c.ldx;
        p.ldc = h.planes * h.dp;
        p.target = c.target;
        p.pos = c.at<int>(h.pos);
        p.count = c.at<int>(h.count);
        p.label = c.at<int>(h.label);
        if (h.backward) {
            p.lse = c.at<float>(h.lse);
            p.factor = c.at<float>(h.factor);
            p.stats = stats;
            p.dloss = dloss_rows;
        }
        p.tokens = h.tokens;
        p.dim = h.dim;
        p.classes = h.classes;
        p.ignore = c.ignore;
        p.rows = h.tokens > HD_COUNTED ? 64 : h.tokens > 4096 ? 8 : 4;
        gathering = cdiv(h.tokens, p.rows);
    }
    if (!gathering && !r.blocks) return RDB_OK;
    if (gathering && h.tokens > HD_COUNTED) {
        int *counts = c.at<int>(h.counts);
        head_count_kernel<<<(unsigned)cdiv(h.tokens, HD_COUNT), 256, 0, c.s>>>(counts, c.target, h.tokens, c.ignore);
        if (int rc = check_launch("head_count_kernel")) return rc;
        p.counts = counts;
    }
    if (h.planes > 1) head_gather_kernel<true><<<(unsigned)(gathering + r.blocks), 256, 0, c.s>>>(p, r, (int)gathering);
    else head_gather_kernel<false><<<(unsigned)(gathering + r.blocks), 256, 0, c.s>>>(p, r, (int)gathering);
    return check_launch("head_gather_kernel");
}

// One block a compute unit where there are no more tiles than that, and stages enough to have two on their way.  us a forward call, two blocks a unit | one: 97 tokens x 640 -> 44480
// 29.1 | 26.6, 717 x 1000 -> 10001 34.6 | 31.9, 2048 x 2048 -> 4000 51.8 | 49.5; 2048 x 256 -> 4000 21.4 | 22.2, 1300 x 64 -> 6000 18.9 | 19.3.
constexpr int HD_SOLO_DIM = 512;
template <bool GRAD> static int head_logits(HeadLogits &p, int64_t classes, bool few, hipStream_t s)
{
    p.tiles_v = (int)cdiv(classes, few ? head_few_tile(classes) : HD_TILE);
    if (few) {
        const unsigned blocks = (unsigned)(GRAD ? p.tiles_v : head_few_blocks(classes));
        if (head_few_tile(classes) == 128) head_logits_few_kernel<GRAD, 128><<<blocks, 256, 0, s>>>(p);
        else head_logits_few_kernel<GRAD, 64><<<blocks, 256, 0, s>>>(p);
        return check_launch(GRAD ? "head_logits_few_kernel<gradient>" : "head_logits_few_kernel");
    }
    const int64_t tiles = p.tiles_v * cdiv(p.tokens, HD_TOK);
    const unsigned blocks = (unsigned)((tiles + 7) / 8 * 8);
    const bool planes = p.plane != 0;
    if (tiles <= num_compute_units() && (planes ? 6 : 1) * p.dim >= HD_SOLO_DIM) {
        if (planes) head_logits_solo_kernel<GRAD, true><<<blocks, 256, 0, s>>>(p);
        else head_logits_solo_kernel<GRAD, false><<<blocks, 256, 0, s>>>(p);
        return check_launch(GRAD ? "head_logits_solo_kernel<gradient>" : "head_logits_solo_kernel");
    }
    if (planes) head_logits_duo_kernel<GRAD, true><<<blocks, 256, 0, s>>>(p);
    else head_logits_duo_kernel<GRAD, false><<<blocks, 256, 0, s>>>(p);
    return check_launch(GRAD ? "head_logits_duo_kernel<gradient>" : "head_logits_duo_kernel");
}

static HeadSum head_sum_of(const HeadCall &c, float *loss, float *stats, int reduction)
{
    const HeadPlan &h = c.h;
    return {reduction == HD_NONE ? nullptr : loss, stats + h.tokens, reduction == HD_NONE ? loss : c.at<float>(h.nll), c.at<unsigned int>(h.count) + 1, c.target, h.tokens, c.ignore,
            reduction == HD_MEAN};
}
static int head_fwd_tiles(const HeadCall &c, float *loss, float *stats, int reduction)
{
    const HeadPlan &h = c.h;
    const bf16_t *w;
    int64_t ldw;
    if (int rc = head_gather(c, nullptr, nullptr, &w, &ldw)) return rc;
    HeadLogits p = {};
    p.x = h.direct ? static_cast<const bf16_t *>(c.x) : c.at<bf16_t>(h.xc);
    p.ldx = h.direct ? c.ldx : h.planes * h.dp;
    p.w = w;
    p.ldw = ldw;
    p.plane = h.planes > 1 ? (int)h.dp : 0;
    p.count = h.direct ? nullptr : c.at<int>(h.count);
    p.cleared = h.direct ? c.at<unsigned int>(h.count) + 1 : nullptr;
    p.dim = (int)h.dp;
    p.classes = (int)h.classes;
    p.part = c.at<float2>(h.part);
    p.picked = c.at<float>(h.picked);
    p.label = h.direct ? nullptr : c.at<int>(h.label);
    p.target = h.direct ? c.target : nullptr;
    p.tokens = h.tokens;
    if (int rc = head_logits<false>(p, h.classes, h.few, c.s)) return rc;
    const HeadMerge m = {stats, p.part, p.picked, h.direct ? nullptr : c.at<int>(h.pos), h.classes, h.parts, head_sum_of(c, loss, stats, reduction)};
    // 16 lanes a token from as many tokens on as give every other compute unit a block of 64
    if (h.tokens >= 8192) head_merge_kernel<16><<<(unsigned)cdiv(h.tokens, 64), 1024, 0, c.s>>>(m);
    else head_merge_kernel<64><<<(unsigned)cdiv(h.tokens, 16), 1024, 0, c.s>>>(m);
    return check_launch("head_merge_kernel");
}
template <typename E> static int head_bwd_tiles(const HeadCall &c, E *dx, E *dw, const float *dloss, const float *stats, int reduction)
{
    const HeadPlan &h = c.h;
    const bf16_t *w;
    int64_t ldw;
    if (int rc = head_gather(c, stats, reduction == HD_NONE ? dloss : nullptr, &w, &ldw)) return rc;
    const HeadScale scale = {reduction == HD_NONE ? nullptr : dloss, reduction == HD_MEAN ? stats + h.tokens : nullptr};
    constexpr bool PLANES = sizeof(E) == 4;
    E *dwc = h.pad_dw && dw ? c.at<E>(h.dw) : dw;
    const int64_t lddw = PLANES ? h.dim : h.dp;
    const int *count = c.at<int>(h.count);
    auto piece = [&](int i) {
        HeadLogits p = {};
        const int64_t v0 = i * h.vp;
        p.x = c.at<bf16_t>(h.xc);
        p.ldx = h.planes * h.dp;
        p.w = w;
        p.ldw = ldw;
        p.plane = PLANES ? (int)h.dp : 0;
        p.plane_g = (int)h.vp;
        p.count = count;
        p.dim = (int)h.dp;
        p.classes = (int)h.classes;
        p.v0 = (int)v0;
        p.tiles_v = (int)cdiv(std::min(h.vp, h.classes - v0), HD_TILE);
        p.tokens = h.tokens;
        p.g = c.at<bf16_t>(h.g) + (i & 1) * h.tokens * h.vp * h.planes;
        p.ldg = h.planes * h.vp;
        p.lse = c.at<float>(h.lse);
        p.factor = c.at<float>(h.factor);
        p.label = c.at<int>(h.label);
        return p;
    };
    HeadLogits p = piece(0);
    if (int rc = head_logits<true>(p, std::min(h.vp, h.classes), h.few, c.s)) return rc;
    auto blocks_of = [](int64_t tiles) { return (int)((tiles + 7) / 8 * 8); };
    for (int i = 0; i < h.pieces; ++i) {
        const int64_t v0 = i * h.vp, n = std::min(h.vp, h.classes - v0);
        HeadProducts q = {};
        q.g = c.at<bf16_t>(h.g) + (i & 1) * h.tokens * h.vp * h.planes;
        q.ldg = h.planes * h.vp;
        q.x = c.at<bf16_t>(h.xc);
        q.ldx = h.planes * h.dp;
        q.plane = (int)h.dp;
        q.plane_g = (int)h.vp;
        q.w = w + v0 * ldw;
        q.ldw = ldw;
        q.count = count;
        q.rows_v = (int)n;
        q.dim = (int)h.dp;
        q.tokens = h.tokens;
        q.tiles_d = (int)cdiv(h.dp, DUO_B);
        q.tiles_v = (int)cdiv(n, HD_TILE);
        q.scale = scale;
        if (dx) {
            q.dx = c.at<float>(h.dx);
            q.lddx = h.dp;
            q.dx_stride = h.tokens * h.dp;
            q.split_v = (int)h.split_v;
            q.splits = (int)cdiv(n, h.split_v);
            q.blocks_dx = blocks_of(q.splits * cdiv(h.tokens, HD_TILE) * q.tiles_d);
        }
        if (dw) {
            q.dw = dwc + v0 * lddw;
            q.lddw = lddw;
            q.blocks_dw = blocks_of((int64_t)q.tiles_v * q.tiles_d);
        }
        HeadLogits next = {};
        int64_t blocks = (int64_t)q.blocks_dw + q.blocks_dx;
        if (i + 1 < h.pieces) {
            next = piece(i + 1);
            blocks += blocks_of(next.tiles_v * cdiv(h.tokens, HD_TOK));
        }
        if (i > 0) head_products_kernel<true, PLANES><<<(unsigned)blocks, 256, 0, c.s>>>(q, next);
        else head_products_kernel<false, PLANES><<<(unsigned)blocks, 256, 0, c.s>>>(q, next);
        if (int rc = check_launch("head_products_kernel")) return rc;
    }
    HeadRepack r = {};
    if constexpr (!PLANES)
        if (dw && h.pad_dw) r = head_repack(dw, dwc, h.dp, h.classes, h.dim);
    const int64_t summing = dx ? std::min<int64_t>(cdiv(h.tokens * h.dp / 4, 256), 8192) : 0;
    if (!summing && !r.blocks) return RDB_OK;
    head_dx_kernel<E><<<(unsigned)(summing + r.blocks), 256, 0, c.s>>>(dx, c.at<float>(h.dx), c.at<int>(h.pos), h.tokens, (int)h.dim, h.dp, h.tokens * h.dp, h.splits, scale, r);
    return check_launch("head_dx_kernel");
}

static HeadRows head_rows(const HeadCall &c)
{
    HeadRows p = {};
    p.logits = c.at<float>(c.h.g);
    p.classes = c.h.classes;
    p.sum.target = c.target;
    p.sum.ignore = c.ignore;
    return p;
}
// logits of classes v0 .. v0 + n
static int head_logits_f32(const HeadCall &c, float *logits, int64_t v0, int64_t n)
{
    const HeadPlan &h = c.h;
    const float *x = static_cast<const float *>(c.x), *w = static_cast<const float *>(c.w) + v0 * c.ldw;
    if (!h.range) return rdb_product_f32(logits, x, c.ldx, 0, w, c.ldw, 0, nullptr, h.tokens, n, h.dim, c.at<void>(h.product), h.product_bytes, c.s);
    const HeadFew p = {x, w, c.ldx, c.ldw, logits, (int)h.tokens, (int)h.dim, (int)n, 0};
    head_few_logits_kernel<<<(unsigned)cdiv(n, 64), 256, 0, c.s>>>(p);
    return check_launch("head_few_logits_kernel");
}
// dx, or what these classes add to it
static int head_dx_f32(const HeadCall &c, float *dx, const float *g, int64_t v0, int64_t n, bool add)
{
    const HeadPlan &h = c.h;
    const float *w = static_cast<const float *>(c.w) + v0 * c.ldw;
    const int64_t count = h.tokens * h.dim;
    if (h.range) {
        const HeadFew p = {g, w, n, c.ldw, c.at<float>(h.dx), (int)h.tokens, (int)h.dim, (int)n, (int)h.range};
        const dim3 grid((unsigned)cdiv(h.dim, 128), (unsigned)cdiv(n, h.range));
        head_few_dx_kernel<<<grid, 256, 0, c.s>>>(p);
        if (int rc = check_launch("head_few_dx_kernel")) return rc;
        head_few_sum_kernel<<<(unsigned)cdiv(count, 256), 256, 0, c.s>>>(dx, p.out, count, (int)grid.y, add);
        return check_launch("head_few_sum_kernel");
    }
    float *to = add ? c.at<float>(h.dx) : dx;
    if (int rc = rdb_product_f32(to, g, n, 0, w, c.ldw, 1, nullptr, h.tokens, h.dim, n, c.at<void>(h.product), h.product_bytes, c.s)) return rc;
    if (!add) return RDB_OK;
    head_add_kernel<<<(unsigned)std::min<int64_t>(cdiv(count, 1024), 4096), 256, 0, c.s>>>(dx, to, count);
    return check_launch("head_add_kernel");
}
static int head_fwd_f32(const HeadCall &c, float *loss, float *stats, float *kept, int reduction)
{
    const HeadPlan &h = c.h;
    HeadRows p = head_rows(c);
    p.state = c.at<float2>(h.part);
    p.picked = c.at<float>(h.picked);
    p.stats = stats;
    p.sum = head_sum_of(c, loss, stats, reduction);
    if (kept) p.logits = kept;
    for (int i = 0; i < h.pieces; ++i) {
        const int64_t v0 = i * h.vp, n = std::min(h.vp, h.classes - v0);
        if (int rc = head_logits_f32(c, p.logits, v0, n)) return rc;
        p.n = (int)n;
        p.v0 = (int)v0;
        p.first = i == 0;
        p.last = i + 1 == h.pieces;
        // a long row in 1024 threads where there are not two rows for every compute unit (15 x 45312: 28 -> 10 us)
        if (h.tokens < 2 * num_compute_units() && n > 4096) head_rows_stats_kernel<1024><<<(unsigned)h.tokens, 1024, 0, c.s>>>(p);
        else head_rows_stats_kernel<256><<<(unsigned)h.tokens, 256, 0, c.s>>>(p);
        if (int rc = check_launch("head_rows_stats_kernel")) return rc;
    }
    if (!p.sum.loss) return RDB_OK;
    head_loss_kernel<<<1, 1024, 0, c.s>>>(p.sum);
    return check_launch("head_loss_kernel");
}
static int head_bwd_f32(const HeadCall &c, float *dx, float *dw, const float *dloss, const float *stats, const float *kept, int reduction)
{
    const HeadPlan &h = c.h;
    HeadRows p = head_rows(c);
    p.stats = const_cast<float *>(stats);
    p.g = p.logits;
    if (kept) p.logits = const_cast<float *>(kept);
    p.scale = {dloss, reduction == HD_MEAN ? stats + h.tokens : nullptr};
    p.dloss = reduction == HD_NONE ? dloss : nullptr;
    p.x = static_cast<const float *>(c.x);
    p.ldx = c.ldx;
    p.dim = (int)h.dim;
    for (int i = 0; i < h.pieces; ++i) {
        const int64_t v0 = i * h.vp, n = std::min(h.vp, h.classes - v0);
        if (!kept)
            if (int rc = head_logits_f32(c, p.logits, v0, n)) return rc;
        p.n = (int)n;
        p.v0 = (int)v0;
        p.xc = dw && i == 0 ? c.at<float>(h.xc) : nullptr;
        p.columns = h.tokens < 2 * num_compute_units() ? 4096 : p.n;
        head_rows_grad_kernel<<<dim3((unsigned)h.tokens, (unsigned)cdiv(n, p.columns)), 256, 0, c.s>>>(p);
        if (int rc = check_launch("head_rows_grad_kernel")) return rc;
        if (dx)
            if (int rc = head_dx_f32(c, dx, p.g, v0, n, i > 0)) return rc;
        if (dw)
            if (int rc = rdb_product_f32(dw + v0 * h.dim, p.g, n, 1, c.at<float>(h.xc), h.dim, 1, nullptr, n, h.dim, h.tokens, c.at<void>(h.product), h.product_bytes, c.s)) return rc;
    }
    return RDB_OK;
}

static int check_head(const char *who, int64_t tokens, int64_t dim, int64_t classes, int dtype, int64_t ldx, int64_t ldw, int reduction)
{
    if (dtype != RDB_BF16 && dtype != RDB_F32) return set_error(RDB_E_DTYPE, "%s: x and w in fp32 or bf16", who);
    if (tokens <= 0 || dim <= 0 || classes <= 0 || classes >= (1ll << 31) - HD_TILE || ldx < dim || ldw < dim || reduction < 0 || reduction > 2)
        return set_error(RDB_E_SHAPE, "%s: bad size %lld x %lld x %lld, leading dimensions %lld and %lld, or reduction %d", who, (long long)tokens, (long long)dim,
                         (long long)classes, (long long)ldx, (long long)ldw, reduction);
    // 32-bit offsets within an operand: x in rows of a multiple of 8 values, a tile of W's rows, a piece of G
    if ((dim + 7) / 8 * 8 * std::max<int64_t>(tokens, HD_TILE) >= (1ll << 29) || tokens >= (1ll << 21) || ldw >= (1ll << 20))
        return set_error(RDB_E_UNSUPPORTED, "%s: x of less than 2^29 values and 2^21 rows, rows of w less than 2^20 apart", who);
    if (cdiv(classes, HD_TILE) * cdiv(tokens, HD_TOK) >= (1ll << 23))   // a launch has less than 2^32 threads
        return set_error(RDB_E_UNSUPPORTED, "%s: less than 2^38 logits", who);
    return RDB_OK;
}

}  // namespace rdb

using namespace rdb;

static HeadPlan head_plan_of(int64_t tokens, int64_t dim, int64_t classes, int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, bool backward, bool want_dx, bool want_dw,
                             bool kept)
{
    const bool whole = dim % 8 == 0;
    return head_plan(tokens, dim, classes, dtype, ldw, backward, want_dx, want_dw, whole && head_aligned(x, ldx, 2) && ldx < (1ll << 20), !whole || !head_aligned(w, ldw, 2), kept);
}

// A product less in a backward pass that few tokens leave bound by the weight: us a step, computed again | kept: 12 tokens x 2048 -> 47643 407 | 306, 69 x 2723 -> 55040 1107 | 862,
// 259 x 3136 -> 96128 5000 | 3960.
extern "C" int64_t rdb_linear_cross_entropy_keeps(int64_t tokens, int64_t dim, int64_t classes, int dtype, int64_t ldw)
{
    if (check_head("rdb_linear_cross_entropy_keeps", tokens, dim, classes, dtype, dim, ldw, 0)) return 0;
    if (dtype != RDB_F32 || !head_keepable(tokens, dim, classes)) return 0;
    return head_plan(tokens, dim, classes, dtype, ldw, true, true, true, false, false, false).pieces == 1 ? tokens * classes : 0;
}

extern "C" int64_t rdb_linear_cross_entropy_workspace_bytes(int64_t tokens, int64_t dim, int64_t classes, int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw,
                                                            int backward, int want_dx, int want_dw)
{
    if (check_head("rdb_linear_cross_entropy_workspace_bytes", tokens, dim, classes, dtype, ldx, ldw, 0)) return 0;
    const bool kept = backward == 2 && rdb_linear_cross_entropy_keeps(tokens, dim, classes, dtype, ldw);
    return head_plan_of(tokens, dim, classes, dtype, x, ldx, w, ldw, backward != 0 && backward != 2, want_dx != 0, want_dw != 0, kept).total;
}

extern "C" int rdb_linear_cross_entropy_fwd(float *loss, float *stats, float *logits, const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype, const int64_t *target,
                                            int64_t tokens, int64_t dim, int64_t classes, int64_t ignore_index, int reduction, void *workspace, int64_t workspace_bytes,
                                            void *stream)
{
    constexpr const char *who = "rdb_linear_cross_entropy_fwd";
    if (int rc = check_head(who, tokens, dim, classes, dtype, ldx, ldw, reduction)) return rc;
    if (!loss || !stats || !x || !w || !target) return set_error(RDB_E_NULL, "%s: an argument is NULL", who);
    if (logits && !rdb_linear_cross_entropy_keeps(tokens, dim, classes, dtype, ldw)) return set_error(RDB_E_UNSUPPORTED, "%s: logits of this size are not kept", who);
    const HeadPlan h = head_plan_of(tokens, dim, classes, dtype, x, ldx, w, ldw, false, false, false, logits != nullptr);
    if (!workspace || workspace_bytes < h.total || ((uintptr_t)workspace & 15)) return set_error(RDB_E_WORKSPACE, "%s: needs %lld bytes from a 16-byte boundary on", who, (long long)h.total);
    const HeadCall c = {h, static_cast<char *>(workspace), x, w, ldx, ldw, target, ignore_index, (hipStream_t)stream};
    return h.tiles ? head_fwd_tiles(c, loss, stats, reduction) : head_fwd_f32(c, loss, stats, logits, reduction);
}

extern "C" int rdb_linear_cross_entropy_bwd(void *dx, void *dw, const float *dloss, const float *stats, const float *logits, const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype,
                                            const int64_t *target, int64_t tokens, int64_t dim, int64_t classes, int64_t ignore_index, int reduction, void *workspace,
                                            int64_t workspace_bytes, void *stream)
{
    constexpr const char *who = "rdb_linear_cross_entropy_bwd";
    if (int rc = check_head(who, tokens, dim, classes, dtype, ldx, ldw, reduction)) return rc;
    if (!dx && !dw) return RDB_OK;
    if (!dloss || !stats || !x || !w || !target) return set_error(RDB_E_NULL, "%s: an argument is NULL", who);
    if (((uintptr_t)dx & 15) || ((uintptr_t)dw & 15)) return set_error(RDB_E_ALIGN, "%s: dx and dw must be 16-byte aligned", who);
    const HeadPlan h = head_plan_of(tokens, dim, classes, dtype, x, ldx, w, ldw, true, dx != nullptr, dw != nullptr, logits != nullptr);
    if (!workspace || workspace_bytes < h.total || ((uintptr_t)workspace & 15)) return set_error(RDB_E_WORKSPACE, "%s: needs %lld bytes from a 16-byte boundary on", who, (long long)h.total);
    if (logits && !rdb_linear_cross_entropy_keeps(tokens, dim, classes, dtype, ldw)) return set_error(RDB_E_UNSUPPORTED, "%s: logits of this size are not kept", who);
    const HeadCall c = {h, static_cast<char *>(workspace), x, w, ldx, ldw, target, ignore_index, (hipStream_t)stream};
    if (!h.tiles) return head_bwd_f32(c, static_cast<float *>(dx), static_cast<float *>(dw), dloss, stats, logits, reduction);
    return dtype == RDB_F32 ? head_bwd_tiles(c, static_cast<float *>(dx), static_cast<float *>(dw), dloss, stats, reduction)
                            : head_bwd_tiles(c, static_cast<bf16_t *>(dx), static_cast<bf16_t *>(dw), dloss, stats, reduction);
}
