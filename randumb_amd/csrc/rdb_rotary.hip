// Rotary positions (modded-nanogpt/gpt_models.py:29-49, with the layouts and frequencies of other models): of a head's first 2 P values,
// pair i at position p becomes (a cos + b sin, b cos - a sin) with the angle p * inv_freq[i] and both factors times `scale`; the
// pairs are values i and P + i, or (interleaved) 2 i and 2 i + 1.  The other values are copied.  The gradient is the same with the sine's sign turned.
//
// Bound by memory: every value is read once and written once, queries and keys in one launch (32768 tokens x 40 heads of 128, bf16: 5.4 TB/s; a large copy: 5.1).  A block takes
// one or a few tokens of one sequence: cosines and sines once a token, into LDS, then 16 bytes a lane and step over all heads.  The angle is formed and reduced to an eighth of
// a turn in 64 bits: at position 10^6 an angle in 32 bits is off by 0.03.
#include "rdb_common.hpp"
#include <algorithm>

namespace rdb {

int num_compute_units();

constexpr int RT_TOKENS = 8;       // at most, of a block
constexpr int RT_PIECES = 192;     // of a block's tokens, about
constexpr int64_t RT_CACHE_BYTES = 256ll << 20;
constexpr int RT_PAIRS = 1024;     // pairs of cosine and sine of a block at most

// n / d for n < 2^31: (n + (n m >> 32)) >> l with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1
struct RtDivide {
    uint32_t d, m;
    int l;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (n + __umulhi(n, m)) >> l; }
};
static RtDivide rt_divide(int64_t d)
{
    RtDivide r = {(uint32_t)d, 0, 0};
    while ((1ll << r.l) < d) ++r.l;
    r.m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << r.l) - (uint64_t)d)) / (uint64_t)d + 1);
    return r;
}
struct RotaryRows {
    void *out;
    const void *in;
    int64_t sb, st, sh;   // elements
    RtDivide heads;
};
struct RotaryParams {
    RotaryRows q, k;      // k.heads.d 0: none
    RtDivide units;       // pieces of a head
    const float *inv_freq;
    const void *positions;
    int64_t pb, pt;       // strides of positions
    int pos_bytes;        // 0: a token's index is its position
    int seq, dim, pairs, tokens, blocks_per_seq;
    int first;            // block of this launch
    bool stream;
    float scale, sign;
};

// N values at once
template <int N> __device__ __forceinline__ void rt_load(float (&v)[N], const float *p) { __builtin_memcpy(v, __builtin_assume_aligned(p, N * 4), N * 4); }
// stream: past the caches (whole pieces of 16 bytes)
template <int N> __device__ __forceinline__ void rt_store(float *p, const float (&v)[N], bool stream)
{
    if constexpr (N == 4)
        if (stream) return store_stream(reinterpret_cast<f32x4 *>(p), f32x4{v[0], v[1], v[2], v[3]});
    __builtin_memcpy(__builtin_assume_aligned(p, N * 4), v, N * 4);
}
template <int N> __device__ __forceinline__ void rt_load(float (&v)[N], const bf16_t *p)
{
    if constexpr (N == 1) {
        v[0] = bf16_to_f32(*p);
    } else {
        uint32_t w[N / 2];
        __builtin_memcpy(w, __builtin_assume_aligned(p, N * 2), N * 2);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            v[2 * e] = lo_f32(w[e]);
            v[2 * e + 1] = hi_f32(w[e]);
        }
    }
}
template <int N> __device__ __forceinline__ void rt_store(bf16_t *p, const float (&v)[N], bool stream)
{
    if constexpr (N == 1) {
        *p = f32_to_bf16(v[0]);
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w[e] = f32x2_to_bf16x2(v[2 * e], v[2 * e + 1]);
        if constexpr (N == 8)
            if (stream) return store_stream(reinterpret_cast<u32x4 *>(p), u32x4{w[0], w[1], w[2], w[3]});
        __builtin_memcpy(__builtin_assume_aligned(p, N * 2), w, N * 2);
    }
}

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

// All heads of a block's tokens, N values (or N of either side of N pairs) a lane and step: rows, strides, the pairs' number and what is behind them are multiples of N.
template <typename E, bool INTERLEAVED, int N>
__device__ __forceinline__ void rt_rows(const RotaryParams &p, const RotaryRows &x, const float2 *cs, int64_t b, int t0, int nt)
{
    constexpr int P = INTERLEAVED ? (N > 1 ? N / 2 : 1) : N;   // pairs of a piece
    const uint32_t paired = (uint32_t)p.pairs / P, total = (uint32_t)nt * x.heads.d * p.units.d;
    const E *in = static_cast<const E *>(x.in) + b * x.sb + (int64_t)t0 * x.st;
    E *out = static_cast<E *>(x.out) + (b * p.seq + t0) * x.heads.d * p.dim;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < total; i += 256) {
        const uint32_t row = p.units(i), u = i - row * p.units.d, t = x.heads(row), h = row - t * x.heads.d;
        const E *src = in + (int64_t)t * x.st + (int64_t)h * x.sh;
        E *dst = out + (int64_t)row * p.dim;
        if (u >= paired) {
            const int c = 2 * p.pairs + (int)(u - paired) * N;
            float a[N];
            rt_load(a, src + c);
            rt_store(dst + c, a, p.stream);
            continue;
        }
        const float2 *w = cs + t * p.pairs + u * P;
        if constexpr (INTERLEAVED && N > 1) {
            float a[N];
            rt_load(a, src + u * N);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float v = a[2 * e];
                a[2 * e] = v * w[e].x + a[2 * e + 1] * w[e].y;
                a[2 * e + 1] = a[2 * e + 1] * w[e].x - v * w[e].y;
            }
            rt_store(dst + u * N, a, p.stream);
        } else {
            const int ia = INTERLEAVED ? 2 * (int)u : (int)u * N, ib = INTERLEAVED ? ia + 1 : p.pairs + ia;
            float a[N], c[N];
            rt_load(a, src + ia);
            rt_load(c, src + ib);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = a[e];
                a[e] = v * w[e].x + c[e] * w[e].y;
                c[e] = c[e] * w[e].x - v * w[e].y;
            }
            rt_store(dst + ia, a, p.stream);
            rt_store(dst + ib, c, p.stream);
        }
    }
}
template <typename E, bool INTERLEAVED, int N> __global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p)
{
    __shared__ float2 cs[RT_PAIRS];
    const int block = p.first + (int)blockIdx.x;
    const int64_t b = block / p.blocks_per_seq;
    const int t0 = (int)(block - b * p.blocks_per_seq) * p.tokens, nt = min(p.tokens, p.seq - t0);
    for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
        const int t = i / p.pairs;
        cs[i] = rt_turn(p, b, t0 + t, i - t * p.pairs);
    }
    __syncthreads();
    rt_rows<E, INTERLEAVED, N>(p, p.q, cs, b, t0, nt);
    if (p.k.heads.d) rt_rows<E, INTERLEAVED, N>(p, p.k, cs, b, t0, nt);
}

// Whether rows may be taken n values at a time.
static bool rt_pieces(const rdb_rotary_rows *x, int es, int n, int64_t batch, int64_t seq)
{
    auto whole = [&](int64_t count, int64_t stride) { return count == 1 || stride % n == 0; };
    return !(((uintptr_t)x->in | (uintptr_t)x->out) & (n * es - 1)) && whole(batch, x->stride_batch) && whole(seq, x->stride_token) && whole(x->heads, x->stride_head);
}
// A launch has less than 2^32 threads.
template <typename E, bool INTERLEAVED, int N> static int launch_rotary(RotaryParams p, int64_t blocks, hipStream_t s)
{
    for (int64_t first = 0; first < blocks; first += 1 << 23) {
        p.first = (int)first;
        rotary_kernel<E, INTERLEAVED, N><<<(unsigned)std::min<int64_t>(blocks - first, 1 << 23), 256, 0, s>>>(p);
        if (int rc = check_launch("rotary_kernel")) return rc;
    }
    return RDB_OK;
}
template <typename E, bool INTERLEAVED> static int launch_rotary(const RotaryParams &p, int64_t blocks, int n, hipStream_t s)
{
    if constexpr (sizeof(E) == 2)
        if (n == 8) return launch_rotary<E, INTERLEAVED, 8>(p, blocks, s);
    if (n == 4) return launch_rotary<E, INTERLEAVED, 4>(p, blocks, s);
    if (n == 2) return launch_rotary<E, INTERLEAVED, 2>(p, blocks, s);
    return launch_rotary<E, INTERLEAVED, 1>(p, blocks, s);
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
    const int es = dtype == RDB_BF16 ? 2 : 4;
    RotaryParams p = {};
    p.q = {q->out, q->in, q->stride_batch, q->stride_token, q->stride_head, rt_divide(q->heads)};
    if (k) p.k = {k->out, k->in, k->stride_batch, k->stride_token, k->stride_head, rt_divide(k->heads)};
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
    int n = 16 / es;   // values a lane takes at once
    while (n > 1 && !(rt_pieces(q, es, n, batch, seq) && (!k || rt_pieces(k, es, n, batch, seq)) && head_dim % n == 0 && (interleaved ? 2 * pairs : pairs) % n == 0)) n /= 2;
    const int64_t paired = interleaved && n > 1 ? 2 * pairs / n : pairs / n;
    p.units = rt_divide(paired + (head_dim - 2 * pairs) / n);
    // A token a block, or as many as give its lanes a piece each or nearly so: what is read and written at a time stays close together.  us with 8 tokens, 2, 1: 32768 tokens x
    // 40 heads of 128 (640 pieces a token) 148, 136, 133; 16384 x 32 x 80, fp32 (640) 67.5, 65.6, 60.4; 8192 x 24 x 64 (96) 10.9 (4 tokens), 10.8, 12.2.
    const int64_t pieces = (q->heads + (k ? k->heads : 0)) * (int64_t)p.units.d;
    int64_t tokens = std::min<int64_t>(RT_TOKENS, std::max<int64_t>(1, RT_PIECES / pieces));
    if (pairs) tokens = std::min<int64_t>(tokens, RT_PAIRS / pairs);
    p.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(tokens, seq));
    // What the last-level cache does not hold goes past it (the first of these 133 -> 123 us); what it holds is for the next launch to find there.
    p.stream = batch * seq * (q->heads + (k ? k->heads : 0)) * head_dim * es > RT_CACHE_BYTES;
    p.blocks_per_seq = (int)cdiv(seq, p.tokens);
    const int64_t blocks = batch * p.blocks_per_seq;
    if (blocks >= (1ll << 31)) return set_error(RDB_E_UNSUPPORTED, "rdb_rotary: too many sequences");
    const auto stream_ = (hipStream_t)stream;
    if (dtype == RDB_BF16) return interleaved ? launch_rotary<bf16_t, true>(p, blocks, n, stream_) : launch_rotary<bf16_t, false>(p, blocks, n, stream_);
    return interleaved ? launch_rotary<float, true>(p, blocks, n, stream_) : launch_rotary<float, false>(p, blocks, n, stream_);
}
