// Rotary positions (modded-nanogpt/gpt_models.py:29-49, with the layouts and frequencies of other models): of a head's first 2 P values,
// pair i at position p becomes (a cos + b sin, b cos - a sin) with the angle p * inv_freq[i] and both factors times `scale`; the
// pairs are values i and P + i, or (interleaved) 2 i and 2 i + 1.  The other values are copied.  The gradient is the same with the sine's sign turned.
//
// Bound by memory: every value is read once and written once, queries and keys in one launch.  A block takes a few tokens of one sequence: cosines and
// sines once a token, into LDS, then 16 bytes a lane and step over all heads.  The angle is formed and reduced to an eighth of
// a turn in 64 bits: at position 10^6 an angle in 32 bits is off by 0.03.
#include "rdb_common.hpp"
#include <algorithm>

namespace rdb {

int num_compute_units();

constexpr int RT_TOKENS = 8;       // at most, of a block
constexpr int RT_PAIRS = 1024;     // pairs of cosine and sine of a block at most

struct RotaryRows {
    void *out;
    const void *in;
    int64_t sb, st, sh;   // elements
    int heads;
};
struct RotaryParams {
    RotaryRows q, k;      // k.heads 0: none
    const float *inv_freq;
    const void *positions;
    int64_t pb, pt;       // strides of positions
    int pos_bytes;        // 0: a token's index is its position
    int seq, dim, pairs, tokens, blocks_per_seq;
    float scale, sign;
};

template <typename E> struct RtPiece;   // 16 bytes as fp32 values
template <> struct RtPiece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void open(float (&v)[4], const u32x4 &w)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    }
    static __device__ __forceinline__ u32x4 close(const float (&v)[4]) { return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}; }
};
template <> struct RtPiece<bf16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void open(float (&v)[8], const u32x4 &w)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = lo_f32(w[e]);
            v[2 * e + 1] = hi_f32(w[e]);
        }
    }
    static __device__ __forceinline__ u32x4 close(const float (&v)[8])
    {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = f32x2_to_bf16x2(v[2 * e], v[2 * e + 1]);
        return w;
    }
};

__device__ __forceinline__ float2 rt_turn(const RotaryParams &p, int64_t b, int t, int i)
{
    int64_t pos = t;
    if (p.pos_bytes == 8) pos = static_cast<const int64_t *>(p.positions)[b * p.pb + t * p.pt];
    else if (p.pos_bytes == 4) pos = static_cast<const int *>(p.positions)[b * p.pb + t * p.pt];
    const double turns = (double)pos * (double)p.inv_freq[i] * 0.15915494309189533577;
    const double quarter = rint(4.0 * turns);
    const float x = 2.0f * (float)(turns - 0.25 * quarter);   // in units of half a turn, at most a quarter
    const int n = (int)(quarter - 4.0 * floor(0.25 * quarter));
    const float c0 = cospif(x), s0 = sinpif(x);
    const float c = n & 1 ? -s0 : c0, s = n & 1 ? c0 : s0;
    return float2{(n & 2 ? -c : c) * p.scale, (n & 2 ? -s : s) * p.scale * p.sign};
}

// Whole pieces of 16 bytes: rows, strides, half the rotary part and the rest are multiples of them.
template <typename E, bool INTERLEAVED> __device__ __forceinline__ void rt_rows(const RotaryParams &p, const RotaryRows &x, const float2 *cs, int64_t b, int t0, int nt)
{
    constexpr int N = RtPiece<E>::N;
    const int paired = INTERLEAVED ? 2 * p.pairs / N : p.pairs / N, units = paired + (p.dim - 2 * p.pairs) / N, per_token = x.heads * units, total = nt * per_token;
    const E *in = static_cast<const E *>(x.in) + b * x.sb + (int64_t)t0 * x.st;
    E *out = static_cast<E *>(x.out) + (b * p.seq + t0) * x.heads * p.dim;
#pragma unroll 4
    for (int i = threadIdx.x; i < total; i += 256) {
        const int row = i / units, u = i - row * units, t = row / x.heads, h = row - t * x.heads;
        const E *src = in + (int64_t)t * x.st + (int64_t)h * x.sh;
        E *dst = out + (int64_t)row * p.dim;
        if (u >= paired) {
            const int c = 2 * p.pairs + (u - paired) * N;
            *reinterpret_cast<u32x4 *>(dst + c) = *reinterpret_cast<const u32x4 *>(src + c);
            continue;
        }
        const float2 *w = cs + t * p.pairs + u * (INTERLEAVED ? N / 2 : N);
        float a[N];
        RtPiece<E>::open(a, *reinterpret_cast<const u32x4 *>(src + u * N));
        if (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const float v = a[2 * e];
                a[2 * e] = v * w[e].x + a[2 * e + 1] * w[e].y;
                a[2 * e + 1] = a[2 * e + 1] * w[e].x - v * w[e].y;
            }
        } else {
            float c[N];
            RtPiece<E>::open(c, *reinterpret_cast<const u32x4 *>(src + p.pairs + u * N));
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = a[e];
                a[e] = v * w[e].x + c[e] * w[e].y;
                c[e] = c[e] * w[e].x - v * w[e].y;
            }
            *reinterpret_cast<u32x4 *>(dst + p.pairs + u * N) = RtPiece<E>::close(c);
        }
        *reinterpret_cast<u32x4 *>(dst + u * N) = RtPiece<E>::close(a);
    }
}
// Any sizes and strides: a pair, or a value of the rest, a lane and step.
template <typename E, bool INTERLEAVED> __device__ __forceinline__ void rt_rows_any(const RotaryParams &p, const RotaryRows &x, const float2 *cs, int64_t b, int t0, int nt)
{
    const int units = p.dim - p.pairs, per_token = x.heads * units, total = nt * per_token;
    const E *in = static_cast<const E *>(x.in) + b * x.sb + (int64_t)t0 * x.st;
    E *out = static_cast<E *>(x.out) + (b * p.seq + t0) * x.heads * p.dim;
#pragma unroll 4
    for (int i = threadIdx.x; i < total; i += 256) {
        const int row = i / units, u = i - row * units, t = row / x.heads, h = row - t * x.heads;
        const E *src = in + (int64_t)t * x.st + (int64_t)h * x.sh;
        E *dst = out + (int64_t)row * p.dim;
        if (u >= p.pairs) {
            dst[p.pairs + u] = src[p.pairs + u];
            continue;
        }
        const int ia = INTERLEAVED ? 2 * u : u, ib = INTERLEAVED ? 2 * u + 1 : p.pairs + u;
        const float2 w = cs[t * p.pairs + u];
        const float a = elem<E>::load(src + ia), c = elem<E>::load(src + ib);
        elem<E>::store(dst + ia, a * w.x + c * w.y);
        elem<E>::store(dst + ib, c * w.x - a * w.y);
    }
}
template <typename E, bool INTERLEAVED, bool PIECES> __global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p)
{
    __shared__ float2 cs[RT_PAIRS];
    const int64_t b = blockIdx.x / p.blocks_per_seq;
    const int t0 = (int)(blockIdx.x - b * p.blocks_per_seq) * p.tokens, nt = min(p.tokens, p.seq - t0);
    for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
        const int t = i / p.pairs;
        cs[i] = rt_turn(p, b, t0 + t, i - t * p.pairs);
    }
    __syncthreads();
    if (PIECES) {
        rt_rows<E, INTERLEAVED>(p, p.q, cs, b, t0, nt);
        if (p.k.heads) rt_rows<E, INTERLEAVED>(p, p.k, cs, b, t0, nt);
    } else {
        rt_rows_any<E, INTERLEAVED>(p, p.q, cs, b, t0, nt);
        if (p.k.heads) rt_rows_any<E, INTERLEAVED>(p, p.k, cs, b, t0, nt);
    }
}

static bool rt_pieces(const rdb_rotary_rows *x, int es)
{
    const int n = 16 / es;
    return !(((uintptr_t)x->in | (uintptr_t)x->out) & 15) && x->stride_batch % n == 0 && x->stride_token % n == 0 && x->stride_head % n == 0;
}
template <typename E> static int launch_rotary(const RotaryParams &p, int64_t blocks, bool pieces, bool interleaved, hipStream_t s)
{
    const dim3 grid((unsigned)blocks);
    if (pieces && interleaved) rotary_kernel<E, true, true><<<grid, 256, 0, s>>>(p);
    else if (pieces) rotary_kernel<E, false, true><<<grid, 256, 0, s>>>(p);
    else if (interleaved) rotary_kernel<E, true, false><<<grid, 256, 0, s>>>(p);
    else rotary_kernel<E, false, false><<<grid, 256, 0, s>>>(p);
    return check_launch("rotary_kernel");
}

}  // namespace rdb

using namespace rdb;

extern "C" int rdb_rotary(const rdb_rotary_rows *q, const rdb_rotary_rows *k, int dtype, int64_t batch, int64_t seq, int64_t head_dim, const float *inv_freq, int64_t pairs,
                          const void *positions, int pos_bytes, int64_t pos_stride_batch, int64_t pos_stride_token, int interleaved, float scale, int inverse, void *stream)
{
    if (dtype != RDB_BF16 && dtype != RDB_F32) return set_error(RDB_E_DTYPE, "rdb_rotary: queries and keys in fp32 or bf16");
    if (!q || (pairs && !inv_freq)) return set_error(RDB_E_NULL, "rdb_rotary: q or inv_freq is NULL");
    if (batch < 0 || seq < 0 || head_dim <= 0 || pairs < 0 || 2 * pairs > head_dim || q->heads < 0 || (k && k->heads < 0))
        return set_error(RDB_E_SHAPE, "rdb_rotary: bad size %lld x %lld x %lld with %lld pairs", (long long)batch, (long long)seq, (long long)head_dim, (long long)pairs);
    if (positions && pos_bytes != 4 && pos_bytes != 8) return set_error(RDB_E_DTYPE, "rdb_rotary: positions of 4 or 8 bytes");
    if (pairs > RT_PAIRS || seq >= (1ll << 31) || head_dim * std::max<int64_t>(q->heads, k ? k->heads : 0) >= (1ll << 27))
        return set_error(RDB_E_UNSUPPORTED, "rdb_rotary: up to %d pairs, 2^31 - 1 tokens and 2^27 values a token", RT_PAIRS);
    if (!q->heads && k) {   // keys alone
        q = k;
        k = nullptr;
    }
    if (!batch || !seq || !q->heads) return RDB_OK;
    if (k && !k->heads) k = nullptr;
    if (!q->in || !q->out || (k && (!k->in || !k->out))) return set_error(RDB_E_NULL, "rdb_rotary: an input or output is NULL");
    const int es = dtype == RDB_BF16 ? 2 : 4, n = 16 / es;
    RotaryParams p = {};
    p.q = {q->out, q->in, q->stride_batch, q->stride_token, q->stride_head, (int)q->heads};
    if (k) p.k = {k->out, k->in, k->stride_batch, k->stride_token, k->stride_head, (int)k->heads};
    p.inv_freq = inv_freq;
    p.positions = positions;
    p.pb = pos_stride_batch;
    p.pt = pos_stride_token;
    p.pos_bytes = positions ? pos_bytes : 0;
    p.seq = (int)seq;
    p.dim = (int)head_dim;
    p.pairs = (int)pairs;
    p.scale = scale;
    p.sign = inverse ? -1.0f : 1.0f;
    // tokens of a block: as many as leave the chip 8 blocks a compute unit
    int64_t tokens = std::min<int64_t>(RT_TOKENS, batch * seq / (8 * num_compute_units()));
    if (pairs) tokens = std::min<int64_t>(tokens, RT_PAIRS / pairs);
    p.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(tokens, seq));
    p.blocks_per_seq = (int)cdiv(seq, p.tokens);
    const int64_t blocks = batch * p.blocks_per_seq;
    if (blocks >= (1ll << 31)) return set_error(RDB_E_UNSUPPORTED, "rdb_rotary: too many sequences");
    const bool pieces = rt_pieces(q, es) && (!k || rt_pieces(k, es)) && head_dim % n == 0 && (interleaved ? 2 * pairs : pairs) % n == 0;
    return dtype == RDB_BF16 ? launch_rotary<bf16_t>(p, blocks, pieces, interleaved != 0, (hipStream_t)stream)
                             : launch_rotary<float>(p, blocks, pieces, interleaved != 0, (hipStream_t)stream);
}
