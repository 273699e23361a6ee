// bf16 matrix products with two blocks on a compute unit: D[a][b] = sum_k A[a][k] * B[b][k] on tiles of 256 x 128, four waves of 128 x 64 in 128 accumulator
// registers each, so that one block's matrix instructions run while the other one is at its epilogue (exponentials, stores of a whole tile) or waits
// for its first operands.  The 256 x 256 tiles of rdb_big.hpp have one block a compute unit and everything behind the main loop comes on top of it.
//
// Operands go from memory straight to LDS (buffer loads with an LDS destination: no registers on the way, which is what leaves room for two blocks), a stage of 64
// contraction values at a time: whole lines of 128 bytes of a row-major matrix.  Half of a compute unit's LDS, 80 KB, holds two stages of A (32 KB
// each) and one of B (16 KB): a wave takes its share of B into registers at the beginning of a stage, and the next stage's B follows into its place.
// An LDS load leaves 64 x 16 bytes in the order of the lanes, so what bank conflicts ask for is done by which 16 bytes of memory a lane asks for.
// Layouts as in rdb_gemm.hpp: K_CONT src[row * ld + k], M_CONT src[k * ld + row] (read by the transposing LDS reads).
#pragma once
#include "rdb_gemm.hpp"

namespace rdb {

constexpr int DUO_A = 256, DUO_B = 128, DUO_K = 64;
constexpr int DUO_MI = 4, DUO_NI = 2;                         // 32 x 32 blocks of a wave
constexpr int DUO_LDS = (2 * DUO_A + DUO_B) * DUO_K, SOLO_LDS = 3 * (DUO_A + DUO_B) * DUO_K;   // elements

// One operand's tile: where its 16-byte pieces lie in LDS, and which of them a lane requests.
template <int ROWS, int LAYOUT> struct DuoOperand {
    static constexpr int ELEMS = ROWS * DUO_K, PER_WAVE = ROWS / 32;   // loads of 1 KB
    i32x4 rsrc;
    uint32_t off, step, advance;   // bytes: this lane's piece 0 at stage 0; from piece to piece; from stage to stage
    int left;                      // K_CONT: stages that hold a value of this lane's
    // A matrix of `rows` rows (M_CONT: columns) and contraction values 0 .. k - 1 (K_CONT: a multiple of 8) from src on.  Rows that are not there come out as zeros or (M_CONT) as
    // what lies behind them inside the matrix: results of their own that nobody stores.  Contraction values from k on are zeros.
    // Less than 2^31 bytes, ld below 2^20.
    __device__ __forceinline__ void set(const bf16_t *src, int64_t ld, int row0, int rows, int k)
    {
        const int t = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
        int64_t bytes;
        if (LAYOUT == K_CONT) {   // rows of 128 bytes, chunk c of row r at position c ^ ((r >> 1) & 7), as OperandTile
            const int row = row0 + wave * 8 + (lane >> 3), chunk = (lane & 7) ^ (((wave & 1) * 4 + (lane >> 4)) & 7);
            off = (uint32_t)(row * ld + chunk * 8) * 2u;
            step = (uint32_t)(32 * ld) * 2u;
            advance = DUO_K * 2u;
            left = (k - chunk * 8 + DUO_K - 1) / DUO_K;
            bytes = rows > 0 && k > 0 ? ((int64_t)(rows - 1) * ld + k) * 2 : 0;
        } else {   // a row for each contraction value k, its 64-byte unit u at position u ^ (k & 3): the four rows of a transposing read cover all banks
            constexpr int PER_K = ROWS / 8, KS = 64 / PER_K;   // pieces of a contraction value, contraction values of a load
            const int kk = wave * KS + lane / PER_K, piece = lane % PER_K, unit = (piece >> 2) ^ (kk & 3);
            off = (uint32_t)(kk * ld + row0 + unit * 32 + (piece & 3) * 8) * 2u;
            step = (uint32_t)(4 * KS * ld) * 2u;
            advance = (uint32_t)(DUO_K * ld) * 2u;
            left = 0x7fffffff;
            bytes = k > 0 ? ((int64_t)(k - 1) * ld + rows) * 2 : 0;
        }
        const uint64_t base = (uint64_t)(uintptr_t)src;
        rsrc = i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)base), __builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32) & 0xffff),
                     __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
    }
    __device__ __forceinline__ uint32_t stage(int s) const { return LAYOUT == K_CONT && s >= left ? BUFFER_OOB * 2 : off + (uint32_t)s * advance; }
    // Requests piece p of the stage that begins at `at` (stage()) into the tile at LDS byte address `to` (this wave's piece 0).
    __device__ __forceinline__ void request(uint32_t at, int p, uint32_t to) const
    {
        const uint32_t o = at + (uint32_t)p * step;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to + (uint32_t)p * 4096u), "v"(o), "s"(rsrc) : "memory");
    }
    // The fragment of 32 rows from rb on, contraction values ks * 16 .. + 15, as OperandTile::frag
    __device__ static __forceinline__ bf16x8 frag(const bf16_t *__restrict__ lds, int rb, int ks, int lane)
    {
        if (LAYOUT == K_CONT) {
            const int r = lane & 31;
            return *reinterpret_cast<const bf16x8 *>(lds + (rb + r) * DUO_K + (((ks * 2 + (lane >> 5)) ^ ((r >> 1) & 7)) * 8));
        } else {
            const int s = lane & 15, k = ks * 16 + (lane >> 5) * 8 + (s >> 2), row = rb + ((lane >> 4) & 1) * 16 + (s & 3) * 4;
            const bf16_t *p = lds + k * ROWS + (((row >> 5) ^ (k & 3)) << 5) + (row & 31);
            Frag8 f;
            f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3))) *)(p));
            f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3))) *)(p + 4 * ROWS));
            return f.v;
        }
    }
};

// The same of an fp32 matrix in three bf16 planes beside each other in its rows (h + m + l of fg_split3, `plane` values apart): the six products of the planes that make an fp32
// one, one after the other, the small ones first.  SIDE 0: A, 1: B of (m m) (l h) (h l) (m h) (h m) (h h).  set() with the whole row, plane 0 first.
template <int ROWS, int LAYOUT, int SIDE> struct DuoPlanes : DuoOperand<ROWS, LAYOUT> {
    int stages;       // of a plane
    uint32_t plane;   // bytes
    __device__ __forceinline__ void set(const bf16_t *src, int64_t ld, int row0, int rows, int k, int plane_values)
    {
        DuoOperand<ROWS, LAYOUT>::set(src, ld, row0, rows, k);
        // all of the last row is in the matrix
        this->rsrc[2] = __builtin_amdgcn_readfirstlane((int)((LAYOUT == K_CONT ? (int64_t)max(rows, 0) * ld : (int64_t)max(k, 0) * ld) * 2));
        stages = max(1, (k + DUO_K - 1) / DUO_K);
        plane = (uint32_t)plane_values * 2u;
    }
    __device__ __forceinline__ uint32_t stage(int s) const
    {
        const int pair = s / stages;
        const uint32_t at = DuoOperand<ROWS, LAYOUT>::stage(s - pair * stages), which = ((SIDE ? 0x121u : 0x49u) >> (2 * min(pair, 6))) & 3u;
        return at + which * plane;
    }
};

__device__ __forceinline__ uint32_t duo_lds_address(const bf16_t *p)
{
    return __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(const bf16_t __attribute__((address_space(3))) *)p);
}

// Contracts `nstage` stages of 64 into acc (at least one: of no contraction values it is a stage of zeros).  lds: DUO_LDS (SOLO_LDS) elements, free on entry and again on return.
// A stage's last k-step waits in registers and is multiplied behind the next barrier, while that stage's first fragments come in (as in big_stage).
// SOLO: one block a compute unit, for launches that have no second one for it: all of LDS holds three stages of both, and two are on their way.
template <bool SOLO, class PA, class PB>
__device__ __forceinline__ void duo_mainloop(f32x16 (&acc)[DUO_MI][DUO_NI], bf16_t *__restrict__ lds, const PA &pa, const PB &pb, int nstage)
{
    const int t = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, arow = (wave >> 1) * DUO_MI * 32, brow = (wave & 1) * DUO_NI * 32;
    constexpr int AHEAD = SOLO ? 2 : 1, BUFFERS = AHEAD + 1;   // stages on their way; of A
    const uint32_t base = duo_lds_address(lds) + (uint32_t)wave * 1024u, b_base = base + BUFFERS * 2u * PA::ELEMS;
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
        const uint32_t at_a = pa.stage(s), at_b = pb.stage(s);
#pragma unroll
        for (int p = 0; p < PA::PER_WAVE; ++p) pa.request(at_a, p, base + s * (2u * PA::ELEMS));
#pragma unroll
        for (int p = 0; p < PB::PER_WAVE; ++p) pb.request(at_b, p, b_base + s * (2u * PB::ELEMS));
    }
    bf16x8 fa[2][DUO_MI], fb[4][DUO_NI];
#pragma unroll
    for (int mi = 0; mi < DUO_MI; ++mi)
#pragma unroll
        for (int e = 0; e < 8; ++e) fa[1][mi][e] = (__bf16)0.0f;
#pragma unroll
    for (int ni = 0; ni < DUO_NI; ++ni)
#pragma unroll
        for (int e = 0; e < 8; ++e) fb[3][ni][e] = (__bf16)0.0f;
    constexpr int N = DUO_MI * DUO_NI;
    auto multiply = [&](int i, int a, int b) { acc[i >> 1][i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[a][i >> 1], fb[b][i & 1], acc[i >> 1][i & 1], 0, 0, 0); };
    int s = 0;
    uint32_t now = 0, then = AHEAD;   // the buffers of stages s and s + AHEAD
    do {
        // stage s has arrived, and nobody reads the buffer of stage s - 1 any more
        if constexpr (SOLO) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PA::PER_WAVE + PB::PER_WAVE) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const bf16_t *As = lds + now * PA::ELEMS, *Bs = lds + BUFFERS * PA::ELEMS + (SOLO ? now * PB::ELEMS : 0u);
        const uint32_t to = base + then * (2u * PA::ELEMS), b_to = b_base + (SOLO ? then * (2u * PB::ELEMS) : 0u), at_a = pa.stage(s + AHEAD), at_b = pb.stage(s + AHEAD);
        now = now == AHEAD ? 0 : now + 1;
        then = then == AHEAD ? 0 : then + 1;
        // Fragments and requests a few in front of each matrix instruction: requests all at once hold a wave up for as long as the compute unit takes to look
        // them up, with its matrix instructions behind them.
#pragma unroll
        for (int i = 0; i < N; ++i) {   // the pending k-step
            if (i == 0) {
                fb[0][0] = PB::frag(Bs, brow, 0, lane);
                fb[0][1] = PB::frag(Bs, brow + 32, 0, lane);
                fa[0][0] = PA::frag(As, arow, 0, lane);
            }
            if (i == 1) {
                fa[0][1] = PA::frag(As, arow + 32, 0, lane);
                fa[0][2] = PA::frag(As, arow + 64, 0, lane);
                fa[0][3] = PA::frag(As, arow + 96, 0, lane);
            }
            if (i == 2 || i == 3) {
                fb[i - 1][0] = PB::frag(Bs, brow, i - 1, lane);
                fb[i - 1][1] = PB::frag(Bs, brow + 32, i - 1, lane);
            }
            if (i >= 4) pa.request(at_a, i - 4, to);
            multiply(i, 1, 3);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {   // k-step 0
            if (i == 0) {
                fb[3][0] = PB::frag(Bs, brow, 3, lane);
                fb[3][1] = PB::frag(Bs, brow + 32, 3, lane);
            }
            if (i == 1 || i == 2) {
                fa[1][2 * i - 2] = PA::frag(As, arow + (2 * i - 2) * 32, 1, lane);
                fa[1][2 * i - 1] = PA::frag(As, arow + (2 * i - 1) * 32, 1, lane);
            }
            if (i >= 3 && i < 7) pa.request(at_a, i + 1, to);
            multiply(i, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!SOLO) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // B is in everybody's registers
#pragma unroll
        for (int i = 0; i < N; ++i) {   // k-step 1
            if (i < PB::PER_WAVE) pb.request(at_b, i, b_to);
            if (i == 1 || i == 2) {
                fa[0][2 * i - 2] = PA::frag(As, arow + (2 * i - 2) * 32, 2, lane);
                fa[0][2 * i - 1] = PA::frag(As, arow + (2 * i - 1) * 32, 2, lane);
            }
            multiply(i, 1, 1);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {   // k-step 2
            if (i == 0 || i == 1) {
                fa[1][2 * i] = PA::frag(As, arow + 2 * i * 32, 3, lane);
                fa[1][2 * i + 1] = PA::frag(As, arow + (2 * i + 1) * 32, 3, lane);
            }
            multiply(i, 0, 2);
            __builtin_amdgcn_sched_barrier(0);
        }
    } while (++s < nstage);
#pragma unroll
    for (int i = 0; i < N; ++i) multiply(i, 1, 3);
    // what was requested past the end has arrived, too, before anybody uses LDS for something else
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ void duo_zero(f32x16 (&acc)[DUO_MI][DUO_NI])
{
#pragma unroll
    for (int mi = 0; mi < DUO_MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < DUO_NI; ++ni) acc[mi][ni] = zero16();
}

}  // namespace rdb
