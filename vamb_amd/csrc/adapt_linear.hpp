// adapt_linear.hpp -- the shared projection with the low-rank adapters of many groups beside it, one launch, gfx950.
//
//   forward   u = x A_g^T            y  = f(x W^T + b + s u B_g^T)
//   backward  v = s (dy f') B_g      dx = (dy f') W + v A_g                (the same kernel on the other orientation: TRANS)
//
// A workgroup of four waves owns BM = 64 MS slots of the row plan (adapt_common.hpp) and BN = 16 NT columns; a wave owns MS
// subtiles of 16 rows, each with one adapter, and all BN columns.  While a K-tile of x and W is in the LDS the wave multiplies its x
// operands with W (NT products) and with its subtiles' A_g (RT = ceil(rank / 16) products, operands straight from memory: they are
// shared by no other wave), so u costs no second pass over x.  Both products are taken as D[column][row]: a
// lane ends with four consecutive columns of one row, and u's accumulator layout (lane: row l & 15, ranks 4 (l >> 4) + i) IS the
// operand layout of the 16-deep product with B_g, which therefore follows without leaving the registers.
//   u is cut into three planes there (24 bits, all of it) for tensors of either type: with two, a bf16 result differed from the rounded exact one
//   in one element of 300 (16 bits of u against the 8 of a rounded sum); the third costs one 16-deep product in three per 16 columns and ranks.
// x reaches the LDS by DMA where its rows are 16-byte aligned bf16, else through registers (any alignment, any row stride; float32 is cut
// into planes there).  The backward pass's p has been cut, masked and brought into the plan's order before (adapt.hip): DMA always.
// LDS rows are 128 B (64 B with three planes); 16-byte pieces are XOR-permuted by the row so that the 16 rows of an operand read fall
// into different bank groups.
#pragma once

#include "adapt_common.hpp"
#include "common.hpp"

#include <type_traits>

namespace vh {
namespace adapt {

// 16 bytes per lane from base + offset to the LDS.  Buffer loads, not global_load_lds: that one is a flat instruction to the compiler, which
// then turns every wait on an LDS read or a register load into a drain of all of them (seen in the ISA: vmcnt(0) in the middle of a
// tile).  An offset at or behind the buffer's end reads zeros.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const void* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void dma16(Buffer b, unsigned offset, unsigned char* lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)lds_wave_base, 16, (int)offset, 0, 0, 0);
}
constexpr unsigned kBehind = 0xfffffff0u;   // behind every buffer (their sizes are below it)
static __device__ const uint4 g_zero32[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};

// ALONE: beside an operand of one plane, which may hold infinities
template <bool ALONE>
__device__ __forceinline__ void cut4(const f32x4 v, s16x4 (&o)[3]) {
    unsigned w[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        unsigned h0, m0, l0, h1, m1, l1;
        split3<ALONE>(v[2 * e], h0, m0, l0);
        split3<ALONE>(v[2 * e + 1], h1, m1, l1);
        if constexpr (ALONE) {
            const unsigned t0 = tiny_of(v[2 * e]), t1 = tiny_of(v[2 * e + 1]);
            m0 = not_zero(m0, t0);
            l0 = not_zero(l0, t0);
            m1 = not_zero(m1, t1);
            l1 = not_zero(l1, t1);
        }
        w[0][e] = (h0 >> 16) | (h1 & 0xffff0000u);
        w[1][e] = (m0 >> 16) | (m1 & 0xffff0000u);
        w[2][e] = (l0 >> 16) | (l1 & 0xffff0000u);
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) o[p] = __builtin_bit_cast(s16x4, u32x2{w[p][0], w[p][1]});
}
__device__ __forceinline__ f32x4 mfma16(s16x4 a, s16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }

// Four elements, `stride` apart, the first `valid` of them (zeros behind): no branch on lanes, what is not there is read from the
// block of zeros.  `vec`: stride 1, and valid is four or none (the same for the whole wave).
__device__ __forceinline__ void load4(const bf16_t* p, int64_t stride, int valid, bool vec, u32x2& o) {
    if (vec) {
        o = (u32x2)*(VH_GLOBAL(u32x2_any, valid >= 4 ? p : (const bf16_t*)g_zero32));
        return;
    }
    bf16_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = *(VH_GLOBAL(bf16_t, i < valid ? p + i * stride : (const bf16_t*)g_zero32));
    o = u32x2{e[0] | (unsigned)e[1] << 16, e[2] | (unsigned)e[3] << 16};
}
__device__ __forceinline__ void load4(const float* p, int64_t stride, int valid, bool vec, f32x4& o) {
    if (vec) {
        o = *(VH_GLOBAL(f32x4_any, valid >= 4 ? p : (const float*)g_zero32));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = *(VH_GLOBAL(float, i < valid ? p + i * stride : (const float*)g_zero32));
}
__device__ __forceinline__ void planes4(const u32x2& r, s16x4 (&o)[1]) { o[0] = __builtin_bit_cast(s16x4, r); }
__device__ __forceinline__ void planes4(const f32x4& r, s16x4 (&o)[3]) { cut4<false>(r, o); }
typedef short tr_s16x4 __attribute__((ext_vector_type(4)));
template <class T> struct Raw4;
template <> struct Raw4<bf16_t> { typedef u32x2 type; };
template <> struct Raw4<float> { typedef f32x4 type; };

// A tile shape: WM x WN waves, each MS x NT subtiles of 16 x 16; two tile buffers of depth BK in the LDS; KG such groups of waves that take
// every KG-th tile of the depth each and add their sums at the end (small grids: more waves a CU to hide each other's latencies).
// NT = 0: only `low` is computed (a backward pass without dx).
template <int WM_, int WN_, int MS_, int NT_, int BK_, int KG_ = 1>
struct Shape {
    static constexpr int WM = WM_, WN = WN_, MS = MS_, NT = NT_, BK = BK_, KG = KG_;
};

// XP: operand planes of x (backward: of p, which for bf16 tensors has two where a slope was applied)
template <class T, class S, int RT, bool TRANS, bool DMA, int XP>
__global__ __launch_bounds__(64 * S::WM * S::WN * S::KG) void linear_kernel(LinArgs a) {
    constexpr int WM = S::WM, WN = S::WN, MS = S::MS, NT = S::NT, NW = WM * WN, THREADS = 64 * NW, KG = S::KG;
    constexpr int P = Elem<T>::planes;
    constexpr int BK = S::BK;
    constexpr int CH = BK / 8;                          // 16-byte pieces of a tile row
    constexpr int BM = 16 * MS * WM, BN = 16 * NT * WN;
    constexpr int XB = BM * BK * 2, WB = BN * BK * 2;   // bytes of a plane
    constexpr int BUF = XP * XB + P * WB;
    constexpr int PX = BM * CH / THREADS;               // x pieces per thread (and plane)
    constexpr int NWI = P * BN * CH / 64;               // W pieces, one wave instruction each
    constexpr int QW = NWI ? (NWI + NW - 1) / NW : 1;
    constexpr int KC = BK / 32;                         // 32-deep products per tile
    constexpr int MU = MS / WN;                         // subtiles whose u this wave computes (its share of the WN waves on the same rows)
    static_assert(PX >= 1 && BM * CH % THREADS == 0 && MS % WN == 0 && (!DMA || TRANS || P == 1) && (!TRANS || DMA) && (TRANS || XP == P), "tile shape");
    static_assert(CH == 4 || CH == 8, "the piece permutations are for these");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

    static_assert(KG == 1 || (WN == 1 && MS == 1), "groups along the depth have narrow waves");
    const int kg = __builtin_amdgcn_readfirstlane((int)threadIdx.x / THREADS), tid = (int)threadIdx.x % THREADS;   // (within the group of waves)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l15 = lane & 15, quad = lane >> 4, wm = wave / WN, wn = wave % WN;
    unsigned char* const tiles = smem + kg * 2 * BUF;
    // workgroup b runs on XCD b % 8: a row tile's column tiles are eight apart, so that XCD's L2 has its x rows after the first
    const int col_tiles = NT ? (a.N + BN - 1) / (BN ? BN : 1) : 1;
    const int bid = blockIdx.x, tile = bid / (8 * col_tiles) * 8 + (bid & 7), n0 = (bid / 8 % col_tiles) * BN;
    const int* slot_row = a.plan + a.ps.o_row;
    const int* sub_group = a.plan + a.ps.o_sub;
    const int K = a.K, r = a.rank, nk = (K + BK - 1) / BK;
    const int n_sub = a.plan[kPlanSubs];

    // 16-byte pieces of a tile row are XOR-permuted by half the row's number within the operand: the 16 rows of an operand read then
    // take the LDS's full 256 B a clock (measured; permuted by a quarter of it, rows of four pieces took 128).  Rows of W are read in
    // another order: a lane's four results of the subtiles 2 i and 2 i + 1 are eight consecutive columns, 32 i + 8 (l15 / 4) + 4 (0 or
    // 1) + l15 % 4 being the column of operand row l15.
    auto swz = [](int row) { return (row >> 1) & (CH - 1); };
    auto swz_w = [](int row) { return ((row >> 1) & 1) | ((row >> 2) & (CH - 2)); };
    auto w_row = [&](int n) { return 32 * (n >> 1) + 8 * (l15 >> 2) + 4 * (n & 1) + (l15 & 3); };

    // ---- x pieces of this thread
    const T* x_src[PX];
    int x_k[PX], rids[PX];
    unsigned x_off[PX];
    Buffer x_buf[XP];
#pragma unroll
    for (int p = 0; p < XP; ++p) {
        if constexpr (TRANS) {
            // the tile's slots follow each other: its own buffer per plane (BM * 2^20 * 2 bytes at most), which ends with the slots
            const int64_t at = (int64_t)tile * BM, left = (a.ps.slots - at) * a.ldx * 2;
            x_buf[p] = buffer_of((const bf16_t*)a.x + ((int64_t)p * a.ps.slots + at) * a.ldx, left > 0 ? (unsigned)min(left, (int64_t)kBehind) : 0u);
        } else {
            x_buf[p] = buffer_of(a.x, a.x_bytes);
        }
    }
#pragma unroll
    for (int q = 0; q < PX && !TRANS; ++q) {
        const int slot = tile * BM + (tid + THREADS * q) / CH;
        rids[q] = slot < (int)a.ps.slots ? slot_row[slot] : -1;   // (slots behind the last run hold anything: n_sub decides below)
    }
    int grp[MU];
#pragma unroll
    for (int m = 0; m < MU; ++m) {
        const int sub = tile * (MS * WM) + wm * MS + wn * MU + m;
        grp[m] = sub < (int)a.ps.subs ? sub_group[sub] : -1;
    }
    int out_row[MS], out_grp[MS];   // this lane's row of the wave's subtiles, and their adapters
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int sub = min(tile * (MS * WM) + wm * MS + m, (int)a.ps.subs - 1);
        out_row[m] = slot_row[16 * sub + l15];
        out_grp[m] = sub_group[sub];
    }
    if (tile * (MS * WM) >= n_sub) return;
#pragma unroll
    for (int m = 0; m < MS; ++m) out_grp[m] = __builtin_amdgcn_readfirstlane(out_grp[m]);
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        const int idx = tid + THREADS * q, row = idx / CH, slot = tile * BM + row;
        x_k[q] = 8 * ((idx % CH) ^ swz(row));
        if constexpr (TRANS) {
            x_off[q] = (unsigned)(row * (int)a.ldx * 2);
        } else {
            const int rid = max(slot < 16 * n_sub ? rids[q] : -1, 0);   // a filling slot takes row 0's values; its results are dropped
            x_src[q] = (const T*)a.x + (int64_t)rid * a.ldx;
            x_off[q] = (unsigned)(rid * a.ldx * (int64_t)sizeof(T));   // (DMA: all of x lies below kBehind)
        }
    }
#pragma unroll
    for (int m = 0; m < MU; ++m) {
        const int sub = tile * (MS * WM) + wm * MS + wn * MU + m;
        grp[m] = __builtin_amdgcn_readfirstlane(sub < n_sub ? grp[m] : -1);
    }

    Raw8<T> x_raw[PX];
    // WHOLE: the tile lies within K (no branch: a wait behind one would drain every load in flight)
    auto fetch_x = [&](auto whole, int k0, unsigned char* buf) {
        if constexpr (DMA) {
#pragma unroll
            for (int p = 0; p < XP; ++p)
#pragma unroll
                for (int q = 0; q < PX; ++q) {
                    const int k = k0 + x_k[q];
                    dma16(x_buf[p], k < K ? x_off[q] + 2 * k : kBehind, buf + p * XB + (wave + NW * q) * 1024);
                }
        } else if constexpr (decltype(whole)::value) {
#pragma unroll
            for (int q = 0; q < PX; ++q) x_raw[q].load(x_src[q] + k0 + x_k[q]);
        } else {
#pragma unroll
            for (int q = 0; q < PX; ++q) x_raw[q] = load8<T>(x_src[q] + k0 + x_k[q], K - k0 - x_k[q]);
        }
    };
    auto keep_x = [&](unsigned char* buf) {
        if constexpr (!DMA) {
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                const Planes8<T> pl = to_planes(x_raw[q]);
#pragma unroll
                for (int p = 0; p < P; ++p) *reinterpret_cast<s16x8*>(buf + p * XB + (tid + THREADS * q) * 16) = pl.p[p];
            }
        }
    };
    // (the workgroup's rows of W begin at a uniform address; within them 32 bits are enough: BN * 2^20 * 2 bytes)
    const Buffer w_buf = buffer_of(a.w + (int64_t)n0 * a.ldw, (unsigned)(2 * (P * a.w_plane - (int64_t)n0 * a.ldw)));
    unsigned w_off[QW];
#pragma unroll
    for (int q = 0; q < QW; ++q) {
        const int idx = (wave + NW * q) * 64 + lane, p = idx / (BN * CH ? BN * CH : 1), rest = idx % (BN * CH ? BN * CH : 1), row = rest / CH;
        w_off[q] = (unsigned)(2 * (p * a.w_plane + (int64_t)row * a.ldw + 8 * ((rest % CH) ^ swz_w(row))));
    }
    auto fetch_w = [&](int k0, unsigned char* buf) {
        if constexpr (NT > 0) {
#pragma unroll
            for (int q = 0; q < QW; ++q)
                if (NWI % NW == 0 || wave + NW * q < NWI) dma16(w_buf, w_off[q] + 2 * k0, buf + (wave + NW * q) * 1024);
        }
    };
    // inner operands: lane = rank l15 (+ 16 j), depth 8 quad ..; what lies outside is read from a block of zeros, so that the loads
    // need no branch (only a ragged last tile of unaligned rows takes the elementwise way)
    const T* in_src[MU][RT];
#pragma unroll
    for (int m = 0; m < MU; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j)
            in_src[m][j] = grp[m] >= 0 && 16 * j + l15 < r ? (const T*)a.inner + ((int64_t)grp[m] * r + 16 * j + l15) * a.ld_inner : nullptr;
    auto fetch_in = [&](auto whole, int k0, Raw8<T> (&in)[MU][KC][RT]) {
        if constexpr (DMA || decltype(whole)::value) {
#pragma unroll
            for (int m = 0; m < MU; ++m)
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int j = 0; j < RT; ++j) {
                        const int k = k0 + 32 * c + 8 * quad;
                        in[m][c][j].load(in_src[m][j] != nullptr && (!DMA || k < K) ? in_src[m][j] + k : (const T*)g_zero32);
                    }
        } else {
#pragma unroll
            for (int m = 0; m < MU; ++m)
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int j = 0; j < RT; ++j) {
                        const int k = k0 + 32 * c + 8 * quad;
                        in[m][c][j] = load8<T>(in_src[m][j] + k, in_src[m][j] != nullptr ? K - k : 0);
                    }
        }
    };

    f32x4 acc[MS][NT ? NT : 1], low[MU][RT];
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < MU; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) low[m][j] = f32x4{0, 0, 0, 0};

    auto compute = [&](const unsigned char* xb, const Raw8<T> (&in)[MU][KC][RT]) {
        const unsigned char* const wb = xb + XP * XB;
        if constexpr (P == 1 && MS == 1 && NT > 0) {
            // one or two products per operand that is read: all reads of the tile go ahead of the products
            s16x8 xa[KC][XP], wa[KC][NT][1];
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int xrow = wm * 16 + l15;
#pragma unroll
                for (int p = 0; p < XP; ++p)
                    xa[c][p] = *reinterpret_cast<const s16x8*>(xb + p * XB + (xrow * CH + ((4 * c + quad) ^ swz(xrow))) * 16);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int row = wn * NT * 16 + w_row(n);
                    wa[c][n][0] = *reinterpret_cast<const s16x8*>(wb + (row * CH + ((4 * c + quad) ^ swz_w(row))) * 16);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < KC; ++c) {
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[0][n] = mma(wa[c][n], xa[c], acc[0][n]);
#pragma unroll
                for (int j = 0; j < RT; ++j) low[0][j] = mma(to_planes(in[0][c][j]).p, xa[c], low[0][j]);
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            s16x8 xf[MS][XP];
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                const int row = (wm * MS + m) * 16 + l15;
#pragma unroll
                for (int p = 0; p < XP; ++p)
                    xf[m][p] = *reinterpret_cast<const s16x8*>(xb + p * XB + (row * CH + ((4 * c + quad) ^ swz(row))) * 16);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s16x8 wf[P];
                const int row = wn * NT * 16 + w_row(n);
#pragma unroll
                for (int p = 0; p < P; ++p)
                    wf[p] = *reinterpret_cast<const s16x8*>(wb + p * WB + (row * CH + ((4 * c + quad) ^ swz_w(row))) * 16);
#pragma unroll
                for (int m = 0; m < MS; ++m) acc[m][n] = mma(wf, xf[m], acc[m][n]);
            }
#pragma unroll
            for (int m = 0; m < MU; ++m)
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const Planes8<T> pl = to_planes(in[m][c][j]);
                    if constexpr (WN == 1) low[m][j] = mma(pl.p, xf[m], low[m][j]);
                    else if (wn == 0) low[m][j] = mma(pl.p, xf[m], low[m][j]);
                    else low[m][j] = mma(pl.p, xf[MS - MU + m], low[m][j]);
                }
        }
    };

    using Yes = std::integral_constant<bool, true>;
    using No = std::integral_constant<bool, false>;
    Raw8<T> in0[MU][KC][RT], in1[MU][KC][RT];
    // Tile kt is multiplied while tile kt + 1 is on its way.  Measured and not kept (524288 x 1024 -> 512, rank 16, when it took 948 us): three and four
    // buffers with counted waits 948, W's operands read three products ahead 949, requests spread between the products 920 -- the
    // loop is not bound by what a tile takes to land, and without any loads it still took 57% of the time.  As it is built, the choice of x's
    // subtiles by `wn` in compute() is four scalar branches in each 32-deep half of a tile, around single products, which part the LDS reads of a
    // half from the products of the one before; 8 waves a CU and these keep the matrix pipe busy for a third of the time.
    auto fetch = [&](int k0, unsigned char* to, Raw8<T> (&in)[MU][KC][RT]) {
        if (k0 + BK <= K) {
            fetch_in(Yes(), k0, in);
            fetch_x(Yes(), k0, to);
        } else {
            fetch_in(No(), k0, in);
            fetch_x(No(), k0, to);
        }
        fetch_w(k0, to + XP * XB);
    };
    if (kg < nk) {
        fetch(kg * BK, tiles, in0);
        keep_x(tiles);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int i = 0; i < (nk + KG - 1) / KG; ++i) {
        const int kt = kg + i * KG;
        unsigned char* const to = tiles + ((i + 1) & 1) * BUF;
        const bool more = kt + KG < nk;
        if (more) fetch((kt + KG) * BK, to, in1);
        __builtin_amdgcn_sched_barrier(0);
        if (KG == 1 || kt < nk) compute(tiles + (i & 1) * BUF, in0);
        __builtin_amdgcn_sched_barrier(0);
        if (more) keep_x(to);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MU; ++m)
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < RT; ++j) in0[m][c][j] = in1[m][c][j];
    }
    if constexpr (KG > 1) {   // the groups' sums, in their order (the tiles are done with)
        f32x4* const part = reinterpret_cast<f32x4*>(smem);   // [KG - 1][NT + RT][THREADS]
        static_assert((KG - 1) * (NT + RT) * THREADS * 16 <= KG * 2 * BUF, "the partial sums fit the tile buffers");
        if (kg > 0) {
            f32x4* const mine = part + (kg - 1) * (NT + RT) * THREADS + tid;
#pragma unroll
            for (int n = 0; n < NT; ++n) mine[n * THREADS] = acc[0][n];
#pragma unroll
            for (int j = 0; j < RT; ++j) mine[(NT + j) * THREADS] = low[0][j];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int q = 0; q < KG - 1; ++q) {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[0][n] += part[(q * (NT + RT) + n) * THREADS + tid];
#pragma unroll
            for (int j = 0; j < RT; ++j) low[0][j] += part[(q * (NT + RT) + NT + j) * THREADS + tid];
        }
    }

    // ---- u of the wave's rows: the WN waves on the same rows computed a share each
    constexpr int LS = 16 * RT + 4;   // floats between rows of the exchange (16-byte pieces of 16 rows in different banks)
    float* const lows = reinterpret_cast<float*>(smem);   // [BM][LS]: the tiles are done with
    static_assert(WN == 1 || BM * LS * 4 <= 2 * BUF, "the exchange fits the tile buffers");
    if constexpr (WN > 1) {
#pragma unroll
        for (int m = 0; m < MU; ++m)
#pragma unroll
            for (int j = 0; j < RT; ++j)
                *reinterpret_cast<f32x4*>(lows + ((wm * MS + wn * MU + m) * 16 + l15) * LS + 16 * j + 4 * quad) = low[m][j];
        __syncthreads();
    }
    typename Raw4<T>::type of[RT][NT ? NT : 1];
    // (behind what other waves may still read: the exchange above, or the groups' sums)
    constexpr int kLows = WN > 1 ? BM * LS * 4 : (KG - 1) * (NT + RT) * THREADS * 16;
    unsigned char* const corner = smem + kLows + wave * 512 * (NT ? NT : 1);   // [16 ranks][16 NT columns]
    static_assert(!(TRANS && P == 1) || kLows + NW * 512 * NT <= KG * 2 * BUF, "the corners fit the tile buffers");
    int have = -1;   // the adapter that `of` holds: neighbouring subtiles mostly have the same
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        if (tile * (MS * WM) + wm * MS + m >= n_sub) break;
        const int g = out_grp[m], rid = out_row[m];
        f32x4 lo[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            if constexpr (WN > 1) lo[j] = *reinterpret_cast<const f32x4*>(lows + ((wm * MS + m) * 16 + l15) * LS + 16 * j + 4 * quad);
            else lo[j] = low[m][j];
            // behind the rank, and in a row without an adapter, stand products with zeros: zero, but NaN where the row holds an infinity or a NaN
#pragma unroll
            for (int i = 0; i < 4; ++i) lo[j][i] = g >= 0 && 16 * j + 4 * quad + i < r ? lo[j][i] : 0.f;
        }
        if (a.low != nullptr && n0 == 0 && wn == 0 && rid >= 0) {
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int rank = 16 * j + 4 * quad;
                float* dst = a.low + (int64_t)rid * r + rank;
                if ((r & 3) == 0 && rank + 4 <= r) {
                    *reinterpret_cast<f32x4*>(dst) = lo[j] * a.low_scale;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (rank + i < r) dst[i] = lo[j][i] * a.low_scale;
                }
            }
        }
        if constexpr (NT > 0) {
            const int nw = n0 + wn * NT * 16;
            if (g >= 0) {
                if constexpr (TRANS && P == 1) {
                    // down [rank][N]: 16 ranks x the wave's columns, 16 bytes at a time, to the wave's own corner of the LDS; the
                    // transposing read gives a lane four ranks of its column
                    if (g != have) {
                        have = g;
                        const T* const base = (const T*)a.outer + (int64_t)g * r * a.N + nw;
#pragma unroll
                        for (int j = 0; j < RT; ++j) {
                            Raw8<T> in[NT / 2];
#pragma unroll
                            for (int q = 0; q < NT / 2; ++q) {
                                const int at = lane + 64 * q, rank = 16 * j + at / (2 * NT), c = 8 * (at % (2 * NT)), left = rank < r ? a.N - nw - c : 0;
                                in[q] = load8<T>(base + (int64_t)min(rank, r - 1) * a.N + c, left);
                            }
#pragma unroll
                            for (int q = 0; q < NT / 2; ++q) *reinterpret_cast<u32x4*>(corner + (lane + 64 * q) * 16) = in[q].v;
                            __builtin_amdgcn_wave_barrier();
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const int c = 32 * (n >> 1) + 8 * (l15 & 3) + 4 * (n & 1);
                                const tr_s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) tr_s16x4*)(corner + (4 * quad + (l15 >> 2)) * NT * 32 + 2 * c));
                                of[j][n] = __builtin_bit_cast(u32x2, t);
                            }
                            __builtin_amdgcn_wave_barrier();
                        }
                    }
                } else if (g != have) {
                    have = g;
#pragma unroll
                    for (int jn = 0; jn < RT * NT; ++jn) {
                        const int n = jn % NT, rank = 16 * (jn / NT) + 4 * quad;
                        const int col = nw + w_row(n);
                        const T* src = (const T*)a.outer + (TRANS ? ((int64_t)g * r + rank) * a.N + col : ((int64_t)g * a.N + col) * r + rank);
                        load4(src, TRANS ? a.N : 1, col < a.N ? r - rank : 0, !TRANS && (r & 3) == 0, of[jn / NT][n]);
                    }
                }
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    s16x4 uf[3];
                    cut4<P == 1>(lo[j] * a.scale, uf);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s16x4 op[P];
                        planes4(of[j][n], op);
#pragma unroll
                        for (int s = 2; s >= 0; --s)
#pragma unroll
                            for (int i = 0; i < P; ++i)
#pragma unroll
                                for (int k = 0; k < 3; ++k)
                                    if (i + k == s) acc[m][n] = mfma16(op[i], uf[k], acc[m][n]);
                    }
                }
            }
            T* yrow = (T*)a.y + (int64_t)max(rid, 0) * a.ldy;
            const bool wide = (a.ldy & 7) == 0 && ((uintptr_t)a.y & 15) == 0;
#pragma unroll
            for (int b = 0; b < NT / 2; ++b) {   // a lane's eight columns of a block of 32
                const int col = nw + 32 * b + 8 * quad;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[m][2 * b + (e >> 2)][e & 3];
                if (!TRANS && a.bias != nullptr) {
                    const f32x4 b0 = *(VH_GLOBAL(f32x4, a.bias + col)), b1 = *(VH_GLOBAL(f32x4, a.bias + col + 4));
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += e < 4 ? b0[e & 3] : b1[e & 3];
                }
                if (!TRANS && a.activation) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = v[e] > 0.f ? v[e] : v[e] * a.slope;
                }
                struct __attribute__((aligned(16))) Row8 { T e[8]; } o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o.e[e] = from_f<T>(v[e]);
                if (rid >= 0) {
                    if (wide && col + 8 <= a.N) {
                        *reinterpret_cast<Row8*>(yrow + col) = o;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e < a.N) yrow[col + e] = o.e[e];
                    }
                }
                if (!TRANS && a.codes != nullptr) {
                    // checkpoint of the rounded y: the block's other columns are in the lanes 16, 32 and 48 further on
                    float amax = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = col + e < a.N ? to_f<T>(o.e[e]) : 0.f;
                        amax = fmaxf(amax, finite_size(v[e]));
                    }
                    amax = fmaxf(amax, __shfl_xor(amax, 16));
                    amax = fmaxf(amax, __shfl_xor(amax, 32));
                    const int k = block_exp(amax);
                    if (rid >= 0 && nw + 32 * b < a.N) {
                        *reinterpret_cast<u32x2*>(a.codes + (int64_t)rid * a.ldc + col) =
                            u32x2{encode4(v[0], v[1], v[2], v[3], k), encode4(v[4], v[5], v[6], v[7], k)};
                        if (quad == 0) a.exps[(int64_t)rid * (a.ldc / kBlockCols) + col / kBlockCols] = (uint8_t)(k + 127);
                    }
                }
            }
        }
    }
}

template <class T, class S, int RT, bool TRANS, bool DMA, int XP>
void launch_one(const LinArgs& a, hipStream_t s) {
    constexpr int P = Elem<T>::planes, BK = S::BK, BM = 16 * S::MS * S::WM, BN = 16 * S::NT * S::WN;
    constexpr int bytes = S::KG * 2 * (XP * BM + P * BN) * BK * 2, threads = 64 * S::WM * S::WN * S::KG;
    static_assert(bytes <= 160 * 1024, "the LDS of a CU");
    const int64_t row_tiles = ceil_div(a.ps.subs, S::MS * S::WM), col_tiles = S::NT ? ceil_div(a.N, BN ? BN : 1) : 1;
    const int64_t blocks = round_up(row_tiles, 8) * col_tiles;
    VH_REQUIRE(fits_a_launch(blocks, threads), "%lld rows of %d columns are too many for one launch", (long long)a.ps.rows, a.N);
    if constexpr (bytes > 65536) {   // per device, cheap, and valid while a stream is captured
        VH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(linear_kernel<T, S, RT, TRANS, DMA, XP>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    }
    linear_kernel<T, S, RT, TRANS, DMA, XP><<<dim3((unsigned)blocks), threads, bytes, s>>>(a);
    VH_HIP(hipGetLastError());
}

template <class T, int RT, bool TRANS, bool DMA, int XP>
void launch_shape(const LinArgs& a, hipStream_t s) {
    constexpr bool F = Elem<T>::planes == 3;
    constexpr int BK = F ? 32 : 64;
    constexpr int KG = RT == 4 ? 2 : 4;   // (rank 33-64: the registers of 16 waves a CU are too few)
    const int tile = linear_tile(a.ps.subs, a.N, F);
    if (a.y == nullptr) {   // (v in the order in which the tile with dx sums it: the adapters' gradients are the same bits with and without dx)
        if constexpr (TRANS) {
            if (tile == kTileNarrow) launch_one<T, Shape<4, 1, 1, 0, BK, KG>, RT, TRANS, DMA, XP>(a, s);
            else launch_one<T, Shape<4, 1, 1, 0, BK, 1>, RT, TRANS, DMA, XP>(a, s);
        }
        return;
    }
    if (tile == kTileNarrow) return launch_one<T, Shape<4, 1, 1, 2, BK, KG>, RT, TRANS, DMA, XP>(a, s);
    if (tile == kTileMid) return launch_one<T, Shape<4, 1, 1, 8, BK>, RT, TRANS, DMA, XP>(a, s);
    if constexpr (!F) {   // 256 rows where the sums fit the registers (65536 rows 512 -> 512, rank 16: 83 us, 91 with 128 rows; rank 32: 183, it spills, 115)
        // and the planes of p the LDS
        if constexpr (RT == 1 && !TRANS) launch_one<T, Shape<4, 2, 4, 8, BK>, RT, TRANS, DMA, XP>(a, s);
        else launch_one<T, Shape<4, 2, 2, 8, BK>, RT, TRANS, DMA, XP>(a, s);
    }
}
template <class T, bool TRANS, bool DMA, int XP>
void launch_rank(const LinArgs& a, hipStream_t s) {
    if (a.rank <= 16) launch_shape<T, 1, TRANS, DMA, XP>(a, s);
    else if (a.rank <= 32) launch_shape<T, 2, TRANS, DMA, XP>(a, s);
    else launch_shape<T, 4, TRANS, DMA, XP>(a, s);
}

}  // namespace adapt
}  // namespace vh
