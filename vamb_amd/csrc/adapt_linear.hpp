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
//   u is cut into planes there (two for bf16 tensors: 16 bits, three for float32), never rounded to 8 bits.
// x reaches the LDS by DMA where its rows are 16-byte aligned, else through registers (any alignment, any row stride; the backward's mask
// is applied there).  LDS rows are 128 B (64 B with three planes); 16-byte pieces are XOR-permuted by the row so that
// the 16 rows of an operand read fall into 16 different bank groups.
#pragma once

#include "adapt_common.hpp"
#include "common.hpp"

namespace vh {
namespace adapt {

__device__ __forceinline__ void dma16(const void* src, unsigned char* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}
static __device__ const uint4 g_zero16 = {0, 0, 0, 0};

template <int PU>
__device__ __forceinline__ void cut4(const f32x4 v, s16x4 (&o)[PU]) {
    unsigned w[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        unsigned h0, m0, l0, h1, m1, l1;
        split3(v[2 * e], h0, m0, l0);
        split3(v[2 * e + 1], h1, m1, l1);
        w[0][e] = (h0 >> 16) | (h1 & 0xffff0000u);
        w[1][e] = (m0 >> 16) | (m1 & 0xffff0000u);
        w[2][e] = (l0 >> 16) | (l1 & 0xffff0000u);
    }
#pragma unroll
    for (int p = 0; p < PU; ++p) o[p] = __builtin_bit_cast(s16x4, u32x2{w[p][0], w[p][1]});
}
__device__ __forceinline__ f32x4 mfma16(s16x4 a, s16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }

// four consecutive elements at p (valid of them) as operand planes
__device__ __forceinline__ void load4_planes(const bf16_t* p, int64_t stride, int valid, s16x4 (&o)[1]) {
    if (stride == 1 && valid >= 4) {
        o[0] = __builtin_bit_cast(s16x4, (u32x2)*reinterpret_cast<const u32x2_any*>(p));
        return;
    }
    s16x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < valid) r[e] = (short)p[e * stride];
    o[0] = r;
}
__device__ __forceinline__ void load4_planes(const float* p, int64_t stride, int valid, s16x4 (&o)[3]) {
    f32x4 r = {0, 0, 0, 0};
    if (stride == 1 && valid >= 4) {
        r = *reinterpret_cast<const f32x4_any*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < valid) r[e] = p[e * stride];
    }
    cut4<3>(r, o);
}

// NT = 0: only `low` is computed (a backward pass without dx)
template <class T, int NT, int MS, int RT, bool TRANS, bool DMA>
__global__ __launch_bounds__(256) void linear_kernel(LinArgs a) {
    constexpr int P = Elem<T>::planes;
    constexpr int PU = P == 1 ? 2 : 3;
    constexpr int BK = P == 1 ? 64 : 32;
    constexpr int CH = BK / 8;                     // 16-byte pieces of a tile row
    constexpr int BM = 64 * MS, BN = 16 * NT;
    constexpr int XB = BM * BK * 2, WB = BN * BK * 2;   // bytes of a plane
    constexpr int BUF = P * (XB + WB);
    constexpr int PX = BM * CH / 256;              // x pieces per thread (and plane)
    constexpr int NWI = P * BN * CH / 64;          // W pieces, one wave instruction each
    constexpr int KC = BK / 32;                    // 32-deep products per tile
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l15 = lane & 15, quad = lane >> 4;
    const int n_sub = a.plan[kPlanSubs];
    const int row_tiles = (n_sub + 4 * MS - 1) / (4 * MS), col_tiles = NT ? (a.N + BN - 1) / (BN ? BN : 1) : 1;
    // workgroup b runs on XCD b % 8: each XCD gets a contiguous run of tiles, the column tiles of a row tile beside each other (its
    // x rows come from that XCD's L2 after the first)
    const int total = row_tiles * col_tiles, xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
    if (local >= (total >> 3) + (xcd < (total & 7))) return;
    const int t = __builtin_amdgcn_readfirstlane(xcd * (total >> 3) + min(xcd, total & 7) + local);
    const int tile = t / col_tiles, n0 = (t % col_tiles) * BN;
    const int* slot_row = a.plan + a.ps.o_row;
    const int* sub_group = a.plan + a.ps.o_sub;
    const int K = a.K, r = a.rank, nk = (K + BK - 1) / BK;

    auto swz = [](int row) { return P == 1 ? ((row >> 1) & 7) : ((row >> 2) & 3); };

    // ---- x pieces of this thread
    const T* x_src[PX];
    const char* m_src[PX];
    int x_k[PX];
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        const int idx = tid + 256 * q, row = idx / CH, slot = tile * BM + row;
        int rid = slot < 16 * n_sub ? slot_row[slot] : -1;
        rid = max(rid, 0);   // a filling slot takes row 0's values; its results are dropped
        x_k[q] = 8 * ((idx % CH) ^ swz(row));
        x_src[q] = (const T*)a.x + (int64_t)rid * a.ldx;
        m_src[q] = a.mask ? (const char*)a.mask + (int64_t)rid * a.ldm * (a.mask_codes ? 1 : (int)sizeof(T)) : nullptr;
    }
    int grp[MS];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int sub = tile * 4 * MS + wave * MS + m;
        grp[m] = __builtin_amdgcn_readfirstlane(sub < n_sub ? sub_group[sub] : -1);
    }

    Raw8<T> x_raw[PX], y_raw[PX];
    u32x2 c_raw[PX];
    auto fetch_x = [&](int k0, unsigned char* buf) {
        if constexpr (DMA) {
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                const int k = k0 + x_k[q];
                dma16(k < K ? (const void*)(x_src[q] + k) : (const void*)&g_zero16, buf + (wave + 4 * q) * 1024);
            }
        } else {
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                const int k = k0 + x_k[q];
                x_raw[q] = load8<T>(x_src[q] + k, K - k);
                if (TRANS && a.mask) {
                    if (a.mask_codes) {
                        c_raw[q] = u32x2{0, 0};
                        if (k < K) c_raw[q] = *reinterpret_cast<const u32x2*>(m_src[q] + k);
                    } else {
                        y_raw[q] = load8<T>((const T*)m_src[q] + k, K - k);
                    }
                }
            }
        }
    };
    auto keep_x = [&](unsigned char* buf) {
        if constexpr (!DMA) {
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                Raw8<T> v = x_raw[q];
                if (TRANS && a.mask) {
                    Raw8<T> o;
                    o.zero();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool pos = a.mask_codes ? !((c_raw[q][e >> 2] >> (8 * (e & 3) + 7)) & 1) : y_raw[q].get(e) > 0.f;
                        const float d = v.get(e);
                        // (bf16: the masked elements are rounded once more, to 8 bits: 2^-9 of terms that the slope made small)
                        o.set(e, from_f<T>(pos ? d : d * a.slope));
                    }
                    v = o;
                }
                const Planes8<T> pl = to_planes(v);
#pragma unroll
                for (int p = 0; p < P; ++p) *reinterpret_cast<s16x8*>(buf + p * XB + (tid + 256 * q) * 16) = pl.p[p];
            }
        }
    };
    auto fetch_w = [&](int k0, unsigned char* buf) {
        if constexpr (NT > 0) {
#pragma unroll
            for (int q = 0; q < (NWI + 3) / 4; ++q) {
                const int wi = wave + 4 * q;
                if (NWI % 4 == 0 || wi < NWI) {
                    const int idx = wi * 64 + lane, p = idx / (BN * CH), rest = idx % (BN * CH), row = rest / CH;
                    dma16(a.w + p * a.w_plane + (int64_t)(n0 + row) * a.ldw + k0 + 8 * ((rest % CH) ^ swz(row)), buf + wi * 1024);
                }
            }
        }
    };
    // A_g operands: lane = rank l15 (+ 16 rt), depth 8 quad ..
    Raw8<T> in_raw[MS][KC][RT];
    auto fetch_in = [&](int k0) {
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const int rank = 16 * j + l15, k = k0 + 32 * c + 8 * quad;
                    const int valid = (grp[m] >= 0 && rank < r) ? K - k : 0;
                    if constexpr (TRANS)
                        in_raw[m][c][j] = load8_strided<T>((const T*)a.inner + ((int64_t)grp[m] * K + k) * r + rank, r, valid);
                    else
                        in_raw[m][c][j] = load8<T>((const T*)a.inner + ((int64_t)grp[m] * r + rank) * K + k, valid);
                }
    };

    f32x4 acc[MS][NT ? NT : 1], low[MS][RT];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < RT; ++j) low[m][j] = f32x4{0, 0, 0, 0};
    }

    unsigned char* const xs0 = smem;
    unsigned char* const ws0 = smem + P * XB;
    fetch_w(0, ws0);
    fetch_x(0, xs0);
    fetch_in(0);
    keep_x(xs0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kt = 0; kt < nk; ++kt) {
        const int cur = kt & 1;
        const unsigned char* const xb = smem + cur * BUF;
        const unsigned char* const wb = xb + P * XB;
        unsigned char* const xn = smem + (cur ^ 1) * BUF;
        const bool more = kt + 1 < nk;
        Planes8<T> in_pl[MS][KC][RT];
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < RT; ++j) in_pl[m][c][j] = to_planes(in_raw[m][c][j]);
        if (more) {
            fetch_w((kt + 1) * BK, xn + P * XB);
            fetch_x((kt + 1) * BK, xn);
            fetch_in((kt + 1) * BK);
        }
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            s16x8 xf[MS][P];
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                const int row = (wave * MS + m) * 16 + l15;
#pragma unroll
                for (int p = 0; p < P; ++p)
                    xf[m][p] = *reinterpret_cast<const s16x8*>(xb + p * XB + (row * CH + ((4 * c + quad) ^ swz(row))) * 16);
            }
#pragma unroll
            for (int m = 0; m < MS; ++m)
#pragma unroll
                for (int j = 0; j < RT; ++j) low[m][j] = mma(in_pl[m][c][j].p, xf[m], low[m][j]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s16x8 wf[P];
                const int row = n * 16 + l15;
#pragma unroll
                for (int p = 0; p < P; ++p)
                    wf[p] = *reinterpret_cast<const s16x8*>(wb + p * WB + (row * CH + ((4 * c + quad) ^ swz(row))) * 16);
#pragma unroll
                for (int m = 0; m < MS; ++m) acc[m][n] = mma(wf, xf[m], acc[m][n]);
            }
        }
        if (more) keep_x(xn);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int slot = tile * BM + (wave * MS + m) * 16 + l15;
        const int rid = slot < 16 * n_sub ? slot_row[slot] : -1;
        if (a.low != nullptr && n0 == 0 && rid >= 0) {
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int rank = 16 * j + 4 * quad;
                float* dst = a.low + (int64_t)rid * r + rank;
                if ((r & 3) == 0 && rank + 4 <= r) {
                    *reinterpret_cast<f32x4*>(dst) = low[m][j] * a.low_scale;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (rank + i < r) dst[i] = low[m][j][i] * a.low_scale;
                }
            }
        }
        if constexpr (NT > 0) {
            if (grp[m] >= 0) {
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    s16x4 uf[PU];
                    cut4<PU>(low[m][j] * a.scale, uf);
                    const int rank = 16 * j + 4 * quad;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int col = n0 + 16 * n + l15;
                        s16x4 of[P];
                        const T* src = (const T*)a.outer + (TRANS ? ((int64_t)grp[m] * r + rank) * a.N + col : ((int64_t)grp[m] * a.N + col) * r + rank);
                        load4_planes(src, TRANS ? a.N : 1, col < a.N ? r - rank : 0, of);
#pragma unroll
                        for (int s = 2; s >= 0; --s)
#pragma unroll
                            for (int i = 0; i < P; ++i)
#pragma unroll
                                for (int k = 0; k < PU; ++k)
                                    if (i + k == s) acc[m][n] = mfma16(of[i], uf[k], acc[m][n]);
                    }
                }
            }
            T* yrow = (T*)a.y + (int64_t)max(rid, 0) * a.ldy;
            const bool wide = (a.ldy & 3) == 0 && ((uintptr_t)a.y & (4 * sizeof(T) - 1)) == 0;
            T out[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = n0 + 16 * n + 4 * quad;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = acc[m][n][i];
                    if (a.bias != nullptr) v += a.bias[col + i];
                    if (a.activation) v = v > 0.f ? v : v * a.slope;
                    out[n][i] = from_f<T>(v);
                }
                if (rid >= 0) {
                    if (wide && col + 4 <= a.N) {
                        struct __attribute__((aligned(4 * sizeof(T)))) Four { T e[4]; };
                        Four f = {{out[n][0], out[n][1], out[n][2], out[n][3]}};
                        *reinterpret_cast<Four*>(yrow + col) = f;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < a.N) yrow[col + i] = out[n][i];
                    }
                }
            }
            if (!TRANS && a.codes != nullptr) {
                // checkpoint of the rounded y: a block of 32 columns is two subtiles, 4 x 2 elements of four lanes
#pragma unroll
                for (int b = 0; b < NT / 2; ++b) {
                    const int c0 = n0 + 32 * b;
                    float v[8], amax = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int col = c0 + 16 * (e >> 2) + 4 * quad + (e & 3);
                        v[e] = col < a.N ? to_f<T>(out[2 * b + (e >> 2)][e & 3]) : 0.f;
                        amax = fmaxf(amax, finite_size(v[e]));
                    }
                    amax = fmaxf(amax, __shfl_xor(amax, 16));
                    amax = fmaxf(amax, __shfl_xor(amax, 32));
                    const int k = block_exp(amax);
                    if (rid >= 0 && c0 < a.N) {
                        uint8_t* dst = a.codes + (int64_t)rid * a.ldc + c0 + 4 * quad;
                        *reinterpret_cast<unsigned*>(dst) = encode4(v[0], v[1], v[2], v[3], k);
                        *reinterpret_cast<unsigned*>(dst + 16) = encode4(v[4], v[5], v[6], v[7], k);
                        if (quad == 0) a.exps[(int64_t)rid * (a.ldc / kBlockCols) + c0 / kBlockCols] = (uint8_t)(k + 127);
                    }
                }
            }
        }
    }
}

template <class T, int NT, int MS, int RT, bool TRANS, bool DMA>
void launch_one(const LinArgs& a, hipStream_t s) {
    constexpr int P = Elem<T>::planes, BK = P == 1 ? 64 : 32;
    constexpr int bytes = 2 * P * (64 * MS + 16 * NT) * BK * 2;
    if constexpr (bytes > 65536) {   // per device, cheap, and valid while a stream is captured
        VH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(linear_kernel<T, NT, MS, RT, TRANS, DMA>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    }
    const int64_t row_tiles = ceil_div(a.ps.subs, 4 * MS), col_tiles = NT ? ceil_div(a.N, 16 * NT) : 1;
    const int64_t blocks = round_up(row_tiles * col_tiles, 8);
    VH_REQUIRE(blocks < (int64_t(1) << 31), "too many rows for one launch");
    linear_kernel<T, NT, MS, RT, TRANS, DMA><<<dim3((unsigned)blocks), 256, bytes, s>>>(a);
    VH_HIP(hipGetLastError());
}

template <class T, int RT, bool TRANS, bool DMA>
void launch_shape(const LinArgs& a, hipStream_t s) {
    if (a.y == nullptr) {
        if constexpr (TRANS) launch_one<T, 0, 1, RT, TRANS, DMA>(a, s);
        return;
    }
    if (a.N <= 32) return launch_one<T, 2, 1, RT, TRANS, DMA>(a, s);
    const int64_t tiles128 = ceil_div(a.ps.subs, 8) * ceil_div(a.N, 128);
    if (tiles128 < 1024) launch_one<T, 8, 1, RT, TRANS, DMA>(a, s);
    else launch_one<T, 8, 2, RT, TRANS, DMA>(a, s);
}
template <class T, bool TRANS, bool DMA>
void launch_rank(const LinArgs& a, hipStream_t s) {
    if (a.rank <= 16) launch_shape<T, 1, TRANS, DMA>(a, s);
    else if (a.rank <= 32) launch_shape<T, 2, TRANS, DMA>(a, s);
    else launch_shape<T, 4, TRANS, DMA>(a, s);
}

}  // namespace adapt
}  // namespace vh
