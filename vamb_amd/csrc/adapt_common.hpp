// adapt_common.hpp -- element types, 8-bit checkpoints and the row plan shared by the adapter kernels (adapt*.hip), gfx950.
//
// Operands of the matrix products.  v_mfma_f32_16x16x32_bf16 is the only matrix instruction of the wide products: bf16 tensors are
// one operand plane, float32 tensors three (x = x0 + x1 + x2, each the next 8 significant bits cut off: exact, 3 x 8 = 24 bits), and of
// the nine products of two such splits the six with i + j <= 2 are taken; the dropped ones (of the product's own sign, as cuts are) are
// below 2^-21 of it together, 2^-24 in the mean.  Six bf16 products run at 2.5 PF / 6 = 420 TF, the fp32 instruction at 157 TF.
//
// 8-bit checkpoints.  One byte per element (e4m3: 1 + 4 + 3 bits) and one exponent byte per 32 columns of a row.  The
// exponent k is the least with amax <= 448 * 2^k, kept in [-117, 120], so that (a) no code saturates, (b) every value code * 2^k has 4
// significant bits and is a normal bf16: the backward products read it without a further rounding.  The sign
// bit is set iff !(x > 0), zeros included: that bit IS the derivative of LeakyReLU, whose argument is positive iff its value is.
// A non-finite element becomes the NaN code (0xff) and does not enter amax.  At k = 120 the code is kept to 240: 256 * 2^120 would be an
// infinity in both types.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vh {
namespace adapt {

typedef unsigned short bf16_t;   // raw bits
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// the same at any element alignment (rows of 107 or 154 columns start anywhere); gfx950 serves unaligned 16-byte loads
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

constexpr int kBlockCols = 32;   // columns that share an exponent
constexpr int kMinExp = -117, kMaxExp = 120;
constexpr int kMaxRank = 64;
constexpr int kMaxGroups = 16384;

template <class T> struct Elem;
template <> struct Elem<bf16_t> { static constexpr int planes = 1; };
template <> struct Elem<float> { static constexpr int planes = 3; };

__device__ __forceinline__ float bf_to_f(bf16_t h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ bf16_t f_to_bf(float x) { return __builtin_bit_cast(bf16_t, (__bf16)x); }   // nearest even

template <class T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<bf16_t>(bf16_t x) { return bf_to_f(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f<bf16_t>(float x) { return f_to_bf(x); }

// (global memory said aloud: a pointer chosen between two objects would be read by flat loads, which also count as LDS accesses)
#define VH_GLOBAL(type, p) (const __attribute__((address_space(1))) type*)(p)

// ---- eight consecutive elements as they were read -------------------------------------------------------------------------
template <class T> struct Raw8;
template <> struct Raw8<bf16_t> {
    u32x4 v;
    __device__ __forceinline__ void zero() { v = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const bf16_t* p) { v = *(VH_GLOBAL(u32x4_any, p)); }
    __device__ __forceinline__ void set(int e, bf16_t x) {   // e: a constant after unrolling; the element's bits are zero before
        v[e >> 1] |= (unsigned)x << (16 * (e & 1));
    }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16)); }
};
template <> struct Raw8<float> {
    f32x4 a, b;
    __device__ __forceinline__ void zero() { a = f32x4{0, 0, 0, 0}; b = a; }
    __device__ __forceinline__ void load(const float* p) {
        a = *(VH_GLOBAL(f32x4_any, p));
        b = *(VH_GLOBAL(f32x4_any, p + 4));
    }
    __device__ __forceinline__ void set(int e, float x) {
        if (e < 4) a[e] = x; else b[e - 4] = x;
    }
    __device__ __forceinline__ float get(int e) const { return e < 4 ? a[e] : b[e - 4]; }
};

// p[0 .. 7], zeros behind the first `valid` (nothing is read behind them)
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int valid) {
    Raw8<T> r;
    r.zero();
    if (valid >= 8) {
        r.load(p);
    } else if (valid > 0) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < valid) r.set(e, *(VH_GLOBAL(T, p + e)));
    }
    return r;
}
// ---- operand planes ---------------------------------------------------------------------------------------------------------
// The three cuts of a float32, for products with three other cuts of which those with i + j <= 2 are taken.  An infinity is +-1, 0, +-inf: its
// last cut meets the other's first alone, which is zero only where the other is zero itself (or below 2^-133), and its first brings
// another infinity's last into the sum; had it been whole in the first, the zero lower cuts of a number such as 0.5 would make a NaN of it.
// A NaN stays one.  WHOLE: an infinity is +-inf, 0, 0, which is less work, for products with one plane that holds none (values of checkpoints;
// 4096 x 1104 x 512: 34.1 us for the gradient of the weight, 35.3 with the other).
template <bool WHOLE = false>
__device__ __forceinline__ void split3(float x, unsigned& h, unsigned& m, unsigned& l) {
    const unsigned b = __float_as_uint(x);
    const bool inf = __builtin_isinf(x);
    if constexpr (WHOLE) {
        h = b & 0xffff0000u;
        const float r = inf ? 0.f : x - __uint_as_float(h);
        m = __float_as_uint(r) & 0xffff0000u;
        l = __float_as_uint(r - __uint_as_float(m));
        return;
    }
    h = inf ? (b & 0x80000000u) | 0x3f800000u : b & 0xffff0000u;
    float r = x - __uint_as_float(h);
    m = inf ? 0u : __float_as_uint(r) & 0xffff0000u;
    const float q = r - __uint_as_float(m);   // at most 8 significant bits: its low half is zero (an infinity: itself)
    l = __float_as_uint(q);
}

// A number's later cut beside an operand of ONE plane, which may hold infinities itself: never zero but for zero, so that the product with an
// infinity is one of the number's sign in every cut.  `tiny` (of `x`'s sign, 2^-126) stands for a zero; it is 2^-25 of x at most: numbers
// below 2^-100 keep their zeros (and make a NaN of an infinity, as if they were zero).  The cut has x's sign or is zero.
__device__ __forceinline__ unsigned tiny_of(float x) {
    return fabsf(x) >= 0x1p-100f ? (__float_as_uint(x) & 0x80000000u) | 0x00800000u : 0u;   // (a NaN: 0)
}
__device__ __forceinline__ unsigned not_zero(unsigned cut, unsigned tiny) { return cut > tiny ? cut : tiny; }   // (bits of one sign: the larger)

template <class T> struct Planes8 { s16x8 p[Elem<T>::planes]; };

__device__ __forceinline__ Planes8<bf16_t> to_planes(const Raw8<bf16_t>& r) {
    Planes8<bf16_t> o;
    o.p[0] = __builtin_bit_cast(s16x8, r.v);
    return o;
}
template <bool WHOLE = false>
__device__ __forceinline__ Planes8<float> to_planes(const Raw8<float>& r) {
    u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned h0, m0, l0, h1, m1, l1;
        split3<WHOLE>(r.get(2 * e), h0, m0, l0);
        split3<WHOLE>(r.get(2 * e + 1), h1, m1, l1);
        w[0][e] = (h0 >> 16) | (h1 & 0xffff0000u);
        w[1][e] = (m0 >> 16) | (m1 & 0xffff0000u);
        w[2][e] = (l0 >> 16) | (l1 & 0xffff0000u);
    }
    Planes8<float> o;
#pragma unroll
    for (int p = 0; p < 3; ++p) o.p[p] = __builtin_bit_cast(s16x8, w[p]);
    return o;
}

// Eight values of p = dy f' as operand planes.  One: they are bf16 as they are (bf16 dy, nothing applied).  Two: bf16 dy with a slope applied, whose
// product has up to 24 bits more than dy; 16 of p's bits are held (the first cut, and the rest rounded to nearest: of one sign, 2^-16 of p
// at most), a plane more than bf16 itself, by which gradients stay as near the exact ones as their own rounding to bf16 lets them (one plane:
// 2^-8, and 1.3 elements in 100 of a gradient differ from the rounded exact one instead of 0.03; the second plane costs 8192 rows 7 us of 53 and
// 65537 rows 60 of 470).  Three: float32.
template <int PP> struct Cut8 { s16x8 p[PP]; };
template <int PP, bool WHOLE = false>
__device__ __forceinline__ Cut8<PP> cut8(const float (&f)[8]) {
    Cut8<PP> o;
    if constexpr (PP == 3) {
        Raw8<float> r;
        r.a = f32x4{f[0], f[1], f[2], f[3]};
        r.b = f32x4{f[4], f[5], f[6], f[7]};
        const Planes8<float> c = to_planes<WHOLE>(r);
#pragma unroll
        for (int p = 0; p < 3; ++p) o.p[p] = c.p[p];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned b = __float_as_uint(f[e]);
            o.p[0][e] = (short)(b >> 16);
            if constexpr (PP == 2) {
                const float r = __builtin_isinf(f[e]) ? 0.f : f[e] - __uint_as_float(b & 0xffff0000u);
                const unsigned low = (unsigned)f_to_bf(r) << 16;
                o.p[1][e] = (short)((WHOLE ? low : not_zero(low, tiny_of(f[e]))) >> 16);
            }
        }
    }
    return o;
}

__device__ __forceinline__ f32x4 mfma32(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfx8, a), __builtin_bit_cast(bfx8, b), c, 0, 0, 0);
}
template <int PA, int PB>
__device__ __forceinline__ f32x4 mma(const s16x8 (&a)[PA], const s16x8 (&b)[PB], f32x4 c) {
#pragma unroll
    for (int s = 2; s >= 0; --s)   // smallest products first
#pragma unroll
        for (int i = 0; i < PA; ++i)
#pragma unroll
            for (int j = 0; j < PB; ++j)
                if (i + j == s) c = mfma32(a[i], b[j], c);
    return c;
}

// ---- 8-bit checkpoints ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.f;   // (a NaN compares false)
}
// least k with amax <= 448 * 2^k (448 = 1.75 * 2^8: the mantissa above 1.75 carries into the exponent), kept in range
__device__ __forceinline__ int block_exp(float amax) {
    const int k = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return min(max(k, kMinExp), kMaxExp);
}
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float((unsigned)(k + 127) << 23); }   // -126 <= k <= 127
// four elements -> four codes
__device__ __forceinline__ unsigned encode4(float x0, float x1, float x2, float x3, int k) {
    const float inv = exp2i(-k), top = k == kMaxExp ? 240.f : 448.f;
    auto y = [&](float x) { return __builtin_amdgcn_fmed3f(x * inv, -top, top); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x0), y(x1), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x2), y(x3), w, true);
    unsigned s = 0, n = 0;
    const float x[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (!(x[e] > 0.f)) s |= 0x80u << (8 * e);
        if (!(fabsf(x[e]) < __builtin_inff())) n |= 0xffu << (8 * e);
    }
    return ((unsigned)w & 0x7f7f7f7fu) | s | n;
}
__device__ __forceinline__ void decode4(unsigned codes, float scale, float (&o)[4]) {   // (the conversion takes the power of two)
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, true);
    o[0] = a[0];
    o[1] = a[1];
    o[2] = b[0];
    o[3] = b[1];
}
__device__ __forceinline__ u32x2 decode4_bf16(unsigned codes, float scale) {   // exact
    return u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
}
// f' of element e from its code: 1, or the slope where the sign bit is set
__device__ __forceinline__ float slope_of(unsigned codes, int e, float slope) {
    const unsigned s = (unsigned)__builtin_amdgcn_sbfe((int)codes, 8 * e + 7, 1);
    return __uint_as_float((s & __float_as_uint(slope)) | (~s & 0x3f800000u));
}

// ---- the row plan -----------------------------------------------------------------------------------------------------------
// Rows sorted by group (stably: sums over a group's rows have one order), every group's run filled up to a multiple of 16 slots, so that
// a 16-row MFMA operand has ONE adapter.  Rows whose group is not in [0, groups) stand last, without an adapter.  An "item" is
// a piece of at most item_rows rows of one group: what a wave of the gradient kernels takes; a group of several items ("multi") writes parts
// that the join kernel adds in their order.  A group without rows has one empty item, which writes its zeros.
struct PlanShape {
    int64_t rows, groups;
    int64_t slots, subs, items, multis, item_rows;
    int64_t o_row, o_sub, o_item, o_multi, words;
};
inline PlanShape plan_shape(int64_t rows, int64_t groups) {
    PlanShape s{};
    s.rows = rows;
    s.groups = groups;
    const int64_t runs = groups + 1 < rows ? groups + 1 : rows;
    s.subs = rows / 16 + runs;
    s.slots = 16 * s.subs;
    int64_t ir = (rows / 512 + 15) / 16 * 16;
    // (few groups: more pieces, many: fewer parts to join.  Gradients and join, 512 + 512 columns, bf16, equal groups, pieces of 128 / 512 rows: 65536 rows of
    // 100 groups 60 / 107 us, 32768 of 50 36 / 45, 2048 of 10 9 / 11; 32768 of 200 45 / 40, 65536 of 300 67 / 60)
    const int64_t least = groups < 128 ? 128 : 512;
    s.item_rows = ir < least ? least : ir;
    s.items = groups + rows / s.item_rows;
    s.multis = rows / s.item_rows + 1;
    s.o_row = 16;
    s.o_sub = s.o_row + s.slots;
    s.o_item = (s.o_sub + s.subs + 3) / 4 * 4;
    s.o_multi = s.o_item + 4 * s.items;
    s.words = s.o_multi + 4 * s.multis;
    return s;
}
// The slot that the gradient kernels read for row i of an item whose rows begin at slot `first`.  Rows behind the item's last are read as that
// one and counted as nothing.  An item without rows has no slot of its own: behind the last run its `first` can be `slots` (one row, whose group
// is not the last: 16 of 16), so the result is kept below it.
__host__ __device__ __forceinline__ int64_t item_slot(int first, int count, int i, int64_t slots) {
    const int last = count > 0 ? count - 1 : 0;
    const int64_t slot = (int64_t)first + (i < last ? i : last);
    return slot < slots ? slot : slots - 1;
}
enum { kPlanSubs = 0, kPlanItems = 1, kPlanMultis = 2, kPlanParts = 3 };

// ---- which kernels a size takes (adapt_linear.hpp: launch_shape; adapt.hip: adapter_grads_rank) -------------------------------------
// Tiles of the projection, kernel times in us.
// Narrow against mid, 512 -> 512, rank 16, 4 groups: bf16 1024 rows (272 narrow workgroups) 11.8 / 11.8, 2048 rows (528) 17.2 / 11.9, 3800 rows
// (960) 24 / 12; float32 22 / 27, 33 / 27, 46 / 28.  One narrow workgroup fills a CU's LDS, so that more than 256 and a few take turns.  Up to 32
// columns three quarters of a mid tile are idle: 512 -> 32, 2048 rows bf16 6.6 / 10.7, float32 12 / 26; 131072 rows 53 / 47 and 115 / 160.
// Mid against wide, bf16: 16000 rows 27.8 / 29.8 (rank 40: 44 / 32), 32768 rows (260 of the 256 x 256) 47.6 / 48.6 (93 / 79), 60000 rows 81 / 62 (152 / 117);
// backward 57 / 57, 102 / 85.  float32 has no wide tile: 128 x 128 took 1.05 of the mid one's time in the mean, and 172 / 155 at 32768 rows.
// Over 150 drawn layers, both directions, this choice takes 1.01 of the fastest tile's time in the mean and 1.36 at worst.
enum { kTileNarrow, kTileMid, kTileWide };   // 64 rows x 32 columns, 64 x 128, and (bf16) 128 or 256 x 256
inline int linear_tile(int64_t subs, int64_t n, bool f32) {
    if (n <= 32 || (subs + 3) / 4 * ((n + 31) / 32) <= 320) return kTileNarrow;
    return f32 || n <= 128 || (subs + 15) / 16 * ((n + 255) / 256) < 256 ? kTileMid : kTileWide;
}
// Waves that share a tile (an item, 128 columns) of the adapters' gradients.  Few tiles: four, so that an item's rows are a quarter of the round
// trips, which is what the largest groups make the launch wait for.  Many, or ranks above 32 (whose sums fill the registers): one, with nothing to add up.
// Groups of unlike sizes (a spread of e^0.5), 8192 rows, 512 + 512 columns, rank 16, bf16, four against one: 50 groups (912 tiles) 13.5 / 20.4 us, 200
// (1728) 15.8 / 22.5 (equal groups: 16.8 / 13.5), 400 (3328) 22.0 / 20.2, 1000 (8128) 41 / 17; float32 4096 rows, rank 8, 50 groups (656) 10.1 / 15.9;
// rank 64, 8620 rows of 11 groups, 256 + 1104 columns (858) 50 / 33.  Over 87 layers this choice takes 1.05 of the faster's time in the mean.
inline int grad_waves(const PlanShape& ps, int64_t n, int64_t k, int64_t rank) {
    return rank <= 32 && ps.items * ((k + 127) / 128 + (n + 127) / 128) < 2048 ? 4 : 1;
}

// ---- arguments of the shared-projection kernel (adapt_linear.hpp) -----------------------------------------------------------------
struct LinArgs {
    const void* x;            // forward: the layer's input [rows][ldx]; backward: p = dy f' as operand planes [planes][slots][ldx], in the plan's order
    int64_t ldx;
    int x_planes;             // backward: p's operand planes
    float slope;
    int activation;           // forward: LeakyReLU(slope) on the result
    const bf16_t* w;          // packed operand [planes][.][ldw]
    int64_t w_plane;          // elements of a plane
    int ldw;
    const float* bias;        // padded (forward)
    const void* inner;        // adapters contracted with x: [groups][rank][ld_inner] (forward: down, backward: up turned around)
    int64_t ld_inner;
    const void* outer;        // adapters of the result (forward: up [groups][N][rank], backward: down [groups][rank][N])
    int K, N, rank;
    float scale, low_scale;   // on the expanded part; on `low` as it is written
    float* low;               // [rows][rank] or nullptr
    void* y;                  // [rows][ldy]; nullptr: only `low` is wanted
    int64_t ldy;
    uint8_t* codes;           // checkpoint of y (nullptr: none), row stride ldc
    int64_t ldc;
    uint8_t* exps;            // row stride ldc / 32
    const int* plan;
    PlanShape ps;
    int dma;                  // forward: x rows are 16-byte aligned, K is a multiple of 8 and x ends below 2^32 - 16 bytes: ...
    unsigned x_bytes;         // ... its size, as a buffer
};
// a launch has fewer than 2^32 threads
inline bool fits_a_launch(int64_t blocks, int64_t threads) { return blocks * threads < (int64_t(1) << 32); }
void launch_linear_bf16(const LinArgs& a, bool backward, hipStream_t s);
void launch_linear_f32(const LinArgs& a, bool backward, hipStream_t s);

}  // namespace adapt
}  // namespace vh
