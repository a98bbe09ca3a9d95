// adapt.hip -- low-rank adapters of many groups of rows beside a shared projection, and 8-bit activation checkpoints: the C entry
// points of include/vambhip.h and every kernel of them but the projection itself (adapt_linear.hpp).  gfx950.
//
// All pointers of these entry points are DEVICE pointers of the calling thread's current device; the calls enqueue on `stream` and
// return; scratch memory is the caller's, so that two streams or two captured graphs never share any.  Nothing is
// allocated, cleared by memset or synchronised.
#include "adapt_common.hpp"
#include "common.hpp"

namespace vh {
namespace adapt {

// =====================================================================================================================
// Row plan: a stable counting sort of the rows by group.  Rows per wave are consecutive; 64 keys at a time are ranked among
// themselves by ballots over the key's bits, the LDS counter of the wave gives the base.
// =====================================================================================================================
__device__ __forceinline__ unsigned long long same_key(int key, int bits) {
    unsigned lo = ~0u, hi = ~0u;
    for (int b = 0; b < bits; ++b) {
        const unsigned s = (unsigned)__builtin_amdgcn_sbfe(key, b, 1);   // all ones where the bit is set
        const unsigned long long v = __ballot(s != 0);
        lo &= ~((unsigned)v ^ s);
        hi &= ~((unsigned)(v >> 32) ^ s);
    }
    return (unsigned long long)hi << 32 | lo;
}
// exclusive scan over a workgroup of 1024; *total = the sum
__device__ __forceinline__ int3 block_scan3(int3 v, int3* total, int* lds /* 3 * 16 */) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int3 s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(s.x, d), y = __shfl_up(s.y, d), z = __shfl_up(s.z, d);
        if (lane >= d) { s.x += x; s.y += y; s.z += z; }
    }
    __syncthreads();
    if (lane == 63) { lds[wave] = s.x; lds[16 + wave] = s.y; lds[32 + wave] = s.z; }
    __syncthreads();
    int3 base = {0, 0, 0}, all = {0, 0, 0};
    for (int w = 0; w < 16; ++w) {
        if (w == wave) base = all;
        all.x += lds[w];
        all.y += lds[16 + w];
        all.z += lds[32 + w];
    }
    *total = all;
    return int3{base.x + s.x - v.x, base.y + s.y - v.y, base.z + s.z - v.z};
}

// One workgroup of 1024: rows per group `count(g)` -> run starts (handed to `start(g, first slot)`); `write`: filling slots, items, multis,
// header.
template <class Count, class Start>
__device__ __forceinline__ void plan_offsets(int* plan, const PlanShape& ps, int* lds, bool write, Count count, Start start) {
    const int G = (int)ps.groups, ir = (int)ps.item_rows;
    int slot0 = 0, item0 = 0, multi0 = 0, part0 = 0;
    for (int base = 0; base <= G; base += 1024) {
        const int g = base + (int)threadIdx.x;
        const int m = g <= G ? count(g) : 0;
        const int filled = (m + 15) & ~15;
        const int pieces = g < G ? max(1, (m + ir - 1) / ir) : 0;
        const int multi = pieces > 1;
        // the two small counts share a word: multis <= rows / item_rows + 1 <= 513, parts <= 2 multis-worth of pieces <= 1100
        int3 total;
        const int3 at = block_scan3(int3{filled, pieces, multi | ((multi ? pieces : 0) << 16)}, &total, lds);
        if (g <= G) {
            const int first = slot0 + at.x;
            start(g, first);
        }
        if (g <= G && write) {
            const int first = slot0 + at.x;
            for (int i = m; i < filled; ++i) plan[ps.o_row + first + i] = -1;
            const int part = part0 + (at.z >> 16);
            for (int i = 0; i < pieces; ++i) {
                int* it = plan + ps.o_item + 4 * (int64_t)(item0 + at.y + i);
                it[0] = g;
                it[1] = first + i * ir;
                it[2] = min(ir, m - i * ir);
                it[3] = multi ? part + i : -1;
            }
            if (multi) {
                int* mu = plan + ps.o_multi + 4 * (int64_t)(multi0 + (at.z & 0xffff));
                mu[0] = g;
                mu[1] = part;
                mu[2] = pieces;
            }
        }
        slot0 += total.x;
        item0 += total.y;
        multi0 += total.z & 0xffff;
        part0 += total.z >> 16;
    }
    if (threadIdx.x == 0 && write) {
        plan[kPlanSubs] = slot0 / 16;
        plan[kPlanItems] = item0;
        plan[kPlanMultis] = multi0;
        plan[kPlanParts] = part0;
    }
}

// 64 PB rows of a wave at a time, their keys requested together: what a key's load takes is paid once per batch
constexpr int PB = 8;
__device__ __forceinline__ void load_keys(const int* groups, int64_t row0, int64_t hi, int G, int (&key)[PB]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < PB; ++b) {
        const int64_t row = row0 + 64 * b + lane;
        key[b] = groups[min(row, hi - 1)];
    }
#pragma unroll
    for (int b = 0; b < PB; ++b) {
        const int64_t row = row0 + 64 * b + lane;
        key[b] = row < hi ? ((unsigned)key[b] < (unsigned)G ? key[b] : G) : G + 1;   // G + 1: no row
    }
}
// (rows that are in the order of their groups already: 64 equal keys are one count and one run of slots)
__device__ __forceinline__ bool all_equal(int key) { return __all(key == __builtin_amdgcn_readfirstlane(key)); }
__device__ __forceinline__ void place_keys(const int (&key)[PB], int64_t row0, int64_t hi, int G, int bits, int* counter, int* plan, const PlanShape& ps) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < PB; ++b) {
        if (row0 + 64 * b >= hi) break;
        const unsigned long long same = all_equal(key[b]) ? ~0ull : same_key(key[b], bits);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (key[b] <= G) {
            const int slot = counter[key[b]] + rank;
            plan[ps.o_row + slot] = (int)(row0 + 64 * b + lane);
            if ((slot & 15) == 0) plan[ps.o_sub + slot / 16] = key[b] < G ? key[b] : -1;
        }
        __builtin_amdgcn_wave_barrier();   // every lane has read its counter (LDS operations of a wave complete in order)
        if (key[b] <= G && rank == 0) counter[key[b]] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}
__device__ __forceinline__ void count_keys(const int (&key)[PB], int G, int* counter) {
#pragma unroll
    for (int b = 0; b < PB; ++b) {
        if (all_equal(key[b])) {
            if ((threadIdx.x & 63) == 0 && key[b] <= G) counter[key[b]] += 64;   // (the wave's own counters)
        } else if (key[b] <= G) {
            atomicAdd(&counter[key[b]], 1);   // integers: any order
        }
    }
}
__device__ __forceinline__ void place_rows(const int* groups, int64_t lo, int64_t hi, int G, int bits, int* counter, int* plan, const PlanShape& ps) {
    for (int64_t row0 = lo; row0 < hi; row0 += 64 * PB) {
        int key[PB];
        load_keys(groups, row0, hi, G, key);
        place_keys(key, row0, hi, G, bits, counter, plan, ps);
    }
}
__device__ __forceinline__ void count_rows(const int* groups, int64_t lo, int64_t hi, int G, int* counter) {
    for (int64_t row0 = lo; row0 < hi; row0 += 64 * PB) {
        int key[PB];
        load_keys(groups, row0, hi, G, key);
        count_keys(key, G, counter);
    }
}

constexpr int kSmallRows = 16384, kSmallCounters = 12 * 1024;   // 48 KB of counters

// Up to 16384 rows, one launch: every workgroup counts ALL rows (their keys come from the L2) and finds the runs' starts for itself, and then
// places its own 1024 rows, 64 a wave.  (One workgroup for all of 8192 rows took 10 us: eight batches of ballots a wave.)
__global__ __launch_bounds__(1024) void plan_small_kernel(const int* groups, int* plan, PlanShape ps, int bits) {
    extern __shared__ int counters[];   // [16][G + 1] of this workgroup's waves, [G + 1] of the rows before it, [G + 1] of all
    __shared__ int lds[48];
    const int G = (int)ps.groups, wave = threadIdx.x >> 6, rows = (int)ps.rows, mine = 1024 * (int)blockIdx.x;
    int* const before = counters + 16 * (G + 1);
    int* const all = before + G + 1;
    for (int i = threadIdx.x; i < 18 * (G + 1); i += 1024) counters[i] = 0;
    __syncthreads();
    int own = G + 1;   // this thread's row of this workgroup
    for (int row0 = 0; row0 < rows; row0 += 1024 * PB) {
        int key[PB];
#pragma unroll
        for (int b = 0; b < PB; ++b) key[b] = groups[min(row0 + 1024 * b + (int)threadIdx.x, rows - 1)];
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            const int first = row0 + 1024 * b, row = first + (int)threadIdx.x;
            if (first >= rows) break;
            const int k = row < rows ? ((unsigned)key[b] < (unsigned)G ? key[b] : G) : G + 1;   // G + 1: no row
            int* const also = first < mine ? before : counters + wave * (G + 1);
            if (all_equal(k)) {   // (sorted rows: 64 additions to one address would be done one by one)
                if ((threadIdx.x & 63) == 0 && k <= G) {
                    atomicAdd(&all[k], 64);
                    if (first <= mine) atomicAdd(&also[k], 64);
                }
            } else if (k <= G) {
                atomicAdd(&all[k], 1);
                if (first <= mine) atomicAdd(&also[k], 1);
            }
            if (first == mine) own = k;
        }
    }
    __syncthreads();
    plan_offsets(plan, ps, lds, blockIdx.x == 0, [&](int g) { return all[g]; },
                 [&](int g, int first) {
                     first += before[g];
                     for (int w = 0; w < 16; ++w) {
                         const int c = counters[w * (G + 1) + g];
                         counters[w * (G + 1) + g] = first;
                         first += c;
                     }
                 });
    __syncthreads();
    const unsigned long long same = all_equal(own) ? ~0ull : same_key(own, bits);
    if (own <= G) {
        const int slot = counters[wave * (G + 1) + own] + __popcll(same & ((1ull << (threadIdx.x & 63)) - 1));
        plan[ps.o_row + slot] = mine + (int)threadIdx.x;
        if ((slot & 15) == 0) plan[ps.o_sub + slot / 16] = own < G ? own : -1;
    }
}

// Larger: one wave per piece of rows; counts [G + 1][pieces], then run totals [G + 1] behind them
__global__ __launch_bounds__(64) void plan_count_kernel(const int* groups, int* scratch, PlanShape ps, int64_t seg, int pieces) {
    extern __shared__ int counters[];
    const int G = (int)ps.groups;
    for (int i = threadIdx.x; i <= G; i += 64) counters[i] = 0;
    __syncthreads();
    const int64_t lo = min(blockIdx.x * seg, ps.rows), hi = min(lo + seg, ps.rows);
    count_rows(groups, lo, hi, G, counters);
    __syncthreads();
    for (int i = threadIdx.x; i <= G; i += 64) scratch[(int64_t)i * pieces + blockIdx.x] = counters[i];
}
__global__ __launch_bounds__(64) void plan_scan_kernel(int* scratch, int G, int pieces) {
    const int g = blockIdx.x, lane = threadIdx.x;
    int* c = scratch + (int64_t)g * pieces;
    int carry = 0;
    for (int i0 = 0; i0 < pieces; i0 += 64) {
        const int i = i0 + lane, v = i < pieces ? c[i] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int u = __shfl_up(s, d);
            if (lane >= d) s += u;
        }
        if (i < pieces) c[i] = carry + s - v;
        carry += __shfl(s, 63);
    }
    if (lane == 0) scratch[(int64_t)(G + 1) * pieces + g] = carry;
}
__global__ __launch_bounds__(1024) void plan_offsets_kernel(int* plan, int* totals, PlanShape ps) {
    __shared__ int lds[48];
    plan_offsets(plan, ps, lds, true, [&](int g) { return totals[g]; }, [&](int g, int first) { totals[g] = first; });
}
__global__ __launch_bounds__(64) void plan_place_kernel(const int* groups, const int* scratch, int* plan, PlanShape ps, int64_t seg, int pieces, int bits) {
    extern __shared__ int counters[];
    const int G = (int)ps.groups;
    for (int i = threadIdx.x; i <= G; i += 64) counters[i] = scratch[(int64_t)(G + 1) * pieces + i] + scratch[(int64_t)i * pieces + blockIdx.x];
    __syncthreads();
    const int64_t lo = min(blockIdx.x * seg, ps.rows), hi = min(lo + seg, ps.rows);
    place_rows(groups, lo, hi, G, bits, counters, plan, ps);
}

static bool plan_is_small(int64_t rows, int64_t groups) { return rows <= kSmallRows && 18 * (groups + 1) <= kSmallCounters; }
static int64_t plan_pieces(int64_t rows) { return rows < 512 ? 1 : (rows / 512 < 1024 ? rows / 512 : 1024); }

// =====================================================================================================================
// Shared weight: both orientations, zero-filled to whole tiles, cut into planes
// =====================================================================================================================
struct WeightShape {
    int64_t np, kp, nq, kq, fwd, bwd, bias_off, bytes;   // fwd: [P][np][kq], bwd: [P][kp][nq]
    int planes;
};
// (a packed orientation stays below 2^32 - 16 bytes, so that its planes are one buffer)
static WeightShape weight_shape(int64_t n, int64_t k, int dtype) {
    WeightShape w{};
    w.planes = dtype == VH_BF16 ? 1 : 3;
    w.np = n <= 128 ? 128 : round_up(n, 256);   // whole result tiles (launch_shape: 256 columns only above 128)
    w.kq = round_up(k, 128);   // the deepest tile
    w.kp = k <= 128 ? 128 : round_up(k, 256);
    w.nq = round_up(n, 128);
    w.fwd = w.np * w.kq;
    w.bwd = w.kp * w.nq;
    w.bias_off = 2 * w.planes * (w.fwd + w.bwd);
    w.bytes = w.bias_off + 4 * w.np;
    VH_REQUIRE(2 * w.planes * (w.fwd > w.bwd ? w.fwd : w.bwd) < 0xfffffff0ll, "a weight of %lld x %lld is too large", (long long)n, (long long)k);
    return w;
}
template <class T>
__global__ __launch_bounds__(256) void pack_weight_kernel(const T* w, int64_t ld, const T* bias, int n, int k, bf16_t* out, float* out_bias, WeightShape ws) {
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    const bool second = i >= ws.fwd;
    const int64_t j = second ? i - ws.fwd : i;
    if (j < (second ? ws.bwd : ws.fwd)) {
        const int64_t stride = second ? ws.nq : ws.kq, a = j / stride, b = j % stride;
        const int64_t row = second ? b : a, col = second ? a : b;
        const bool in = row < n && col < k;
        bf16_t* dst = out + (second ? ws.planes * ws.fwd : 0) + j;
        const int64_t plane = second ? ws.bwd : ws.fwd;
        if constexpr (sizeof(T) == 2) {
            dst[0] = in ? w[row * ld + col] : (T)0;
        } else {
            unsigned h, m, l;
            split3(in ? w[row * ld + col] : 0.f, h, m, l);
            dst[0] = (bf16_t)(h >> 16);
            dst[plane] = (bf16_t)(m >> 16);
            dst[2 * plane] = (bf16_t)(l >> 16);
        }
    }
    if (i < ws.np) out_bias[i] = bias != nullptr && i < n ? to_f<T>(bias[i]) : 0.f;
}

// =====================================================================================================================
// Checkpoints
// =====================================================================================================================
// Four lanes share a block of 32 columns, eight each.  Bound by memory: 1000003 x 512 bf16 in 372 us, 4.1 TB/s of the 4.9 that a large copy
// reaches; the way back (codes to bf16) in 297 us, 5.2 TB/s.
template <class T>
__global__ __launch_bounds__(256) void checkpoint_kernel(const T* x, int64_t ldx, int64_t rows, int cols, uint8_t* codes, uint8_t* exps) {
    const int chunks = (cols + kBlockCols - 1) / kBlockCols * 4;
    const int64_t total = rows * chunks;
    const int64_t first = blockIdx.x * (int64_t)256 + threadIdx.x, step = (int64_t)gridDim.x * 256;   // multiples of four: a block's lanes stay together
    for (int64_t i = first; i < total; i += step) {
        const int64_t row = i / chunks;
        const int ch = (int)(i - row * chunks);
        const Raw8<T> v = load8<T>(x + row * ldx + 8 * ch, cols - 8 * ch);
        float f[8], amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = v.get(e);
            amax = fmaxf(amax, finite_size(f[e]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const int k = block_exp(amax);
        const u32x2 o = {encode4(f[0], f[1], f[2], f[3], k), encode4(f[4], f[5], f[6], f[7], k)};
        *reinterpret_cast<u32x2*>(codes + 8 * i) = o;   // codes are dense: [rows][8 * chunks]
        if ((ch & 3) == 0) exps[i >> 2] = (uint8_t)(k + 127);
    }
}
template <class T>
__global__ __launch_bounds__(256) void restore_kernel(const uint8_t* codes, const uint8_t* exps, int64_t rows, int cols, T* out) {
    const int chunks = (cols + kBlockCols - 1) / kBlockCols * 4;
    const int64_t total = rows * chunks, step = (int64_t)gridDim.x * 256;
    const bool wide = cols % 8 == 0 && (uintptr_t)out % 16 == 0;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / chunks;
        const int c0 = 8 * (int)(i - row * chunks);
        const u32x2 w = *reinterpret_cast<const u32x2*>(codes + 8 * i);
        const float scale = __uint_as_float((unsigned)exps[i >> 2] << 23);
        float f[8];
        decode4(w[0], scale, reinterpret_cast<float(&)[4]>(f[0]));
        decode4(w[1], scale, reinterpret_cast<float(&)[4]>(f[4]));
        T* dst = out + row * cols + c0;
        if (wide && c0 + 8 <= cols) {
            struct __attribute__((aligned(16))) Eight { T e[8]; };
            Eight o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.e[e] = from_f<T>(f[e]);
            *reinterpret_cast<Eight*>(dst) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e < cols) dst[e] = from_f<T>(f[e]);
        }
    }
}

// A tensor that a backward pass reads: elements of T, or checkpoint codes
struct Source {
    const void* p;         // elements or codes
    const uint8_t* exps;   // nullptr: elements
    int64_t ld;            // in elements / bytes
};
template <class T>
struct Eight {             // eight columns of a row as read
    Raw8<T> raw;
    u32x2 code;
    unsigned exp;
};
template <class E>
__device__ __forceinline__ void read_codes8(const Source& s, int64_t row, int col, int valid, E& o) {
    o.code = u32x2{0, 0};
    o.exp = 0;
    if (valid > 0) {   // rows are filled up to a multiple of 32 codes (of value zero)
        o.code = *(VH_GLOBAL(u32x2, (const uint8_t*)s.p + row * s.ld + col));
        o.exp = *(VH_GLOBAL(uint8_t, s.exps + row * (s.ld / kBlockCols) + col / kBlockCols));
    }
}
template <class T>
__device__ __forceinline__ void read8(const Source& s, int64_t row, int col, int valid, Eight<T>& o) {
    if (s.exps == nullptr) o.raw = load8<T>((const T*)s.p + row * s.ld + col, valid);
    else read_codes8(s, row, col, valid, o);
}
template <class T>
__device__ __forceinline__ void values8(const Source& s, const Eight<T>& v, float (&f)[8]) {
    if (s.exps == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v.raw.get(e);
    } else {
        const float scale = __uint_as_float(v.exp << 23);
        decode4(v.code[0], scale, reinterpret_cast<float(&)[4]>(f[0]));
        decode4(v.code[1], scale, reinterpret_cast<float(&)[4]>(f[4]));
    }
}
// the first n of eight neighbouring results (at any alignment)
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
    if (n >= 8) {
        if constexpr (sizeof(T) == 2) {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = f_to_bf(v[2 * e]) | (unsigned)f_to_bf(v[2 * e + 1]) << 16;
            *reinterpret_cast<u32x4_any*>(p) = o;
        } else {
            *reinterpret_cast<f32x4_any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_any*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = from_f<T>(v[e]);
    }
}
template <class T>
__device__ __forceinline__ void store4(T* p, f32x4 v, int n) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<u32x2_any*>(p) = u32x2{f_to_bf(v[0]) | (unsigned)f_to_bf(v[1]) << 16, f_to_bf(v[2]) | (unsigned)f_to_bf(v[3]) << 16};
        else
            *reinterpret_cast<f32x4_any*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = from_f<T>(v[i]);
    }
}
// f'(y) of eight columns applied to f
template <class T>
__device__ __forceinline__ void masked8(const Source& s, const Eight<T>& v, float slope, float (&f)[8]) {
    if (s.exps != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= slope_of(v.code[e >> 2], e & 3, slope);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v.raw.get(e) > 0.f ? f[e] : f[e] * slope;
    }
}

// =====================================================================================================================
// Gradients of the adapters:  down_g = sum v^T x  [rank][K],  up_g = s sum p^T u  [N][rank]
// One wave = one item (at most item_rows rows of one group) and 128 columns of x or of p.  v_mfma_f32_16x16x4_f32: its operands
// are one element per lane, so eight consecutive columns that a lane has read are the operands of eight instructions and nothing is
// transposed; products and sums are fp32 whatever the tensors' type.  65537 rows of 1000 groups, rank 32, 1104 + 512 columns, bf16: 136 us for
// 6.8 GF (50 TF of the 157 that the instruction has; the rows of a group are few steps, whose latency is what counts) and 100 MB of gradients.
// =====================================================================================================================
struct AdapterGradArgs {
    Source x, mask;            // mask.p == nullptr: f' = 1
    const void* dy;
    int64_t ldy;
    const float* low;          // u [rows][rank], from the forward pass
    const float* v;            // [rows][rank], s included
    void *ddown, *dup;
    const void* up;            // [groups][N][rank], and ...
    void* turned;              // ... [groups][rank][ldp], zeros behind N
    bf16_t* p;                 // dy f' as operand planes [PP][slots][ldp] in the plan's order, zeros behind N and in filling slots
    int64_t ldp;
    float* parts;
    int K, N, rank;
    float scale, slope;
    const int* plan;
    PlanShape ps;
};

// An item's rows, 4 H a step, and 128 columns: one wave (SPLIT = 1), or the workgroup's four, each with every fourth step (SPLIT = 4; their
// sums are added in order).  PP: p's planes.  WHOLE: all columns exist, so that the loads need no branch.
template <class T, int RT, int H, int SPLIT, int PP, bool UP, bool WHOLE>
__device__ __forceinline__ void adapter_grad_tile(const AdapterGradArgs& a, const int* it, int tile0, f32x4 (*red)[8][64]) {
    const int g = it[0], first = it[1], count = it[2], part = it[3];
    const int* slot_row = a.plan + a.ps.o_row;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, quad = lane >> 4;
    const int C = UP ? a.N : a.K, c0 = tile0 + 8 * l15, valid = WHOLE ? 8 : C - c0, r = a.rank;
    const float* small = UP ? a.low : a.v;
    constexpr int PW = UP ? PP : 1;
    const int begin = SPLIT > 1 ? 4 * H * wave : 0;
    constexpr int STEP = 4 * H * SPLIT;

    f32x4 acc[RT][8];
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[j][e] = f32x4{0, 0, 0, 0};

    Eight<T> w[H];           // of x ...
    s16x8 wp[H][PW];         // ... or of p's planes, which stand in the plan's order
    float s[H][RT];
    auto row_of = [&](int i) { return i < count ? slot_row[first + i] : -1; };
    auto fetch = [&](const int (&rid)[H], int i) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int row = max(rid[h], 0);   // (a row that is not there is read as row 0 and counts with a factor of zero ...)
            if constexpr (UP) {
                const int64_t slot = item_slot(first, count, i + quad + 4 * h, a.ps.slots), at = min((int64_t)c0, a.ldp - 8);   // (in bounds; not used behind N)
#pragma unroll
                for (int p = 0; p < PW; ++p)
                    wp[h][p] = __builtin_bit_cast(s16x8, *(VH_GLOBAL(u32x4, a.p + ((int64_t)p * a.ps.slots + slot) * a.ldp + at)));
            } else {
                read8<T>(a.x, row, c0, valid, w[h]);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) s[h][j] = small[(int64_t)row * r + min(16 * j + l15, r - 1)];
        }
    };
    int rid[H], nxt[H];
#pragma unroll
    for (int h = 0; h < H; ++h) rid[h] = row_of(begin + quad + 4 * h);
#pragma unroll
    for (int h = 0; h < H; ++h) nxt[h] = row_of(begin + STEP + quad + 4 * h);
    fetch(rid, begin);
    for (int i = begin; i < count; i += STEP) {
        float f[H][8], sc[H][RT];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if constexpr (UP) {   // (the cuts add up to what they were cut from)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[h][e] = bf_to_f((bf16_t)wp[h][PW - 1][e]);
#pragma unroll
                    for (int p = PW - 2; p >= 0; --p) f[h][e] += bf_to_f((bf16_t)wp[h][p][e]);
                }
            } else {
                values8<T>(a.x, w[h], f[h]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[h][e] = rid[h] >= 0 ? f[h][e] : 0.f;   // (... on zeros: row 0 may hold anything)
#pragma unroll
            for (int j = 0; j < RT; ++j) sc[h][j] = rid[h] >= 0 && 16 * j + l15 < r ? s[h][j] : 0.f;
            rid[h] = nxt[h];
        }
        if (i + STEP < count) {
            fetch(rid, i + STEP);
#pragma unroll
            for (int h = 0; h < H; ++h) nxt[h] = row_of(i + 2 * STEP + quad + 4 * h);
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(sc[h][j], f[h][e], acc[j][e], 0, 0, 0);
    }
    if constexpr (SPLIT > 1) {
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            if (j) __syncthreads();
            if (wave > 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) red[wave - 1][e][lane] = acc[j][e];
            }
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[j][e] += red[0][e][lane] + red[1][e][lane] + red[2][e][lane];
            }
        }
        if (wave > 0) return;
    }
    const int64_t pair = (int64_t)r * (a.K + a.N);
    float* po = part >= 0 ? a.parts + part * pair + (UP ? (int64_t)r * a.K : 0) : nullptr;
    T* dst = UP ? (T*)a.dup + (int64_t)g * a.N * r : (T*)a.ddown + (int64_t)g * r * a.K;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        const int rank = 16 * j + 4 * quad;
        if constexpr (UP) {   // up [N][rank]: four ranks of each of eight columns
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int n = e < valid ? r - rank : 0;
                const int64_t at = (int64_t)(c0 + e) * r + rank;
                const f32x4 v = acc[j][e] * a.scale;
                if (po) store4<float>(po + at, v, n);
                else store4<T>(dst + at, v, n);
            }
        } else {              // down [rank][K]: eight columns of each of four ranks
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[j][e][i];   // (v has the scale)
                const int n = rank + i < r ? valid : 0;
                const int64_t at = (int64_t)(rank + i) * a.K + c0;
                if (po) store8<float>(po + at, v, n);
                else store8<T>(dst + at, v, n);
            }
        }
    }
}
// up [N][rank] of an adapter that some row asks for -> [rank][N], the orientation that dy is contracted with: the projection reads
// its inner operands 16 bytes at a time along the depth.  64 columns, all ranks.
template <class T>
__device__ __forceinline__ void turn_up(const AdapterGradArgs& a, int item, int n0, T* tile /* [64][rank | 1] */) {
    if (item >= a.plan[kPlanItems]) return;
    const int* it = a.plan + a.ps.o_item + 4 * (int64_t)item;
    if (it[2] == 0 || (item > 0 && it[-4] == it[0])) return;   // no rows; a later piece of the same group
    const int r = a.rank, pitch = r | 1, n = min(64, a.N - n0), tid = threadIdx.x;
    const T* src = (const T*)a.up + (int64_t)it[0] * a.N * r + (int64_t)n0 * r;   // n * rank neighbouring elements
    T* out = (T*)a.turned + (int64_t)it[0] * a.ldp * r + n0;
    for (int i = 8 * tid; i < n * r; i += 8 * 256) {
        const Raw8<T> v = load8<T>(src + i, n * r - i);
        int c = i / r, j = i - c * r;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (i + e < n * r) tile[c * pitch + j] = from_f<T>(v.get(e));
            if (++j == r) { j = 0; ++c; }
        }
    }
    __syncthreads();
    for (int i = tid; i < 8 * r; i += 256) {
        const int j = i >> 3, c = 8 * (i & 7);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < n ? to_f<T>(tile[(c + e) * pitch + j]) : 0.f;
        if (n0 + c < a.ldp) store8<T>(out + (int64_t)j * a.ldp + c, v, 8);   // (ldp is a multiple of 8)
    }
}
// p = dy f'(y), cut into operand planes (cut8), in the plan's order
template <class T, int PP>
__device__ __forceinline__ void mask_and_order(const AdapterGradArgs& a, int64_t chunk0) {
    const int per = (int)(a.ldp / 8);
    const int slots = 16 * a.plan[kPlanSubs];
    const Source dy = {a.dy, nullptr, a.ldy};
    constexpr int Q = 4;   // pieces of eight columns a thread, requested together
    int64_t slot[Q];
    int col[Q], rid[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int64_t i = chunk0 + threadIdx.x + 256 * q;
        slot[q] = i / per;
        col[q] = 8 * (int)(i - slot[q] * per);
        rid[q] = a.plan[a.ps.o_row + min(slot[q], (int64_t)slots - 1)];
    }
    Eight<T> w[Q], m[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        read8<T>(dy, max(rid[q], 0), col[q], a.N - col[q], w[q]);
        if (a.mask.p != nullptr) read8<T>(a.mask, max(rid[q], 0), col[q], a.N - col[q], m[q]);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (slot[q] >= slots) continue;
        float f[8];
        values8<T>(dy, w[q], f);
        if (a.mask.p != nullptr) masked8<T>(a.mask, m[q], a.slope, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rid[q] >= 0 ? f[e] : 0.f;
        const Cut8<PP> pl = cut8<PP>(f);
#pragma unroll
        for (int p = 0; p < PP; ++p)
            *reinterpret_cast<s16x8*>(a.p + ((int64_t)p * a.ps.slots + slot[q]) * a.ldp + col[q]) = pl.p[p];
    }
}
// before the projection's pass, two kinds of workgroups: up turned around (64 columns each), and p
template <class T, int PP>
__global__ __launch_bounds__(256) void adapter_first_kernel(AdapterGradArgs a) {
    __shared__ T tile[64 * (kMaxRank + 1)];
    const int turns = (a.N + 63) / 64;
    const int64_t b = blockIdx.x, turning = a.ps.items * turns;
    if (b < turning) turn_up<T>(a, (int)(b / turns), 64 * (int)(b % turns), tile);
    else mask_and_order<T, PP>(a, (b - turning) * 1024);
}
// behind it (v): tiles of down, then tiles of up
template <class T, int RT, int H, int SPLIT, int PP>
__global__ __launch_bounds__(256) void adapter_grad_kernel(AdapterGradArgs a) {
    __shared__ f32x4 red[SPLIT > 1 ? 3 : 1][SPLIT > 1 ? 8 : 1][64];
    auto* const r = reinterpret_cast<f32x4(*)[8][64]>(red);
    if ((int)blockIdx.x >= a.plan[kPlanItems]) return;
    const int* it = a.plan + a.ps.o_item + 4 * (int64_t)blockIdx.x;
    const int downs = (a.K + 127) / 128, ups = (a.N + 127) / 128;
    int tile = SPLIT > 1 ? (int)blockIdx.y : 4 * (int)blockIdx.y + ((int)threadIdx.x >> 6);
    if (tile < downs) {
        if (128 * tile + 128 <= a.K) adapter_grad_tile<T, RT, H, SPLIT, PP, false, true>(a, it, 128 * tile, r);
        else adapter_grad_tile<T, RT, H, SPLIT, PP, false, false>(a, it, 128 * tile, r);
    } else if ((tile -= downs) < ups) {
        if (128 * tile + 128 <= a.N) adapter_grad_tile<T, RT, H, SPLIT, PP, true, true>(a, it, 128 * tile, r);
        else adapter_grad_tile<T, RT, H, SPLIT, PP, true, false>(a, it, 128 * tile, r);
    }
}
template <class T>
__global__ __launch_bounds__(256) void adapter_join_kernel(AdapterGradArgs a) {
    if ((int)blockIdx.y >= a.plan[kPlanMultis]) return;
    const int* mu = a.plan + a.ps.o_multi + 4 * (int64_t)blockIdx.y;
    const int g = mu[0], part = mu[1], n = mu[2];
    const int64_t half = (int64_t)a.rank * a.K, pair = (int64_t)a.rank * (a.K + a.N);
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (i >= pair) return;
    float s = 0.f;
    for (int p = 0; p < n; ++p) s += a.parts[(part + p) * pair + i];
    if (i < half) ((T*)a.ddown)[(int64_t)g * half + i] = from_f<T>(s);
    else ((T*)a.dup)[(int64_t)g * a.N * a.rank + i - half] = from_f<T>(s);
}

// =====================================================================================================================
// Few rows: no plan.  A workgroup = 16 rows x 16 columns; eight waves share the depth of the projection and, one distinct adapter at a
// time, the u of the rows; the last 256 products with B_g are plain fused multiply-adds in float32.  One row, 304 -> 512, rank 8, bf16: 4.6 us,
// of which a launch is 4.  Every workgroup reads the rows' adapters: rows x rank x K decides when the plan and the projection behind it are
// faster (vamb_amd/adapters.py).
// =====================================================================================================================
struct FewArgs {
    const void* x;
    int64_t ldx;
    const int* groups;
    const bf16_t* w;
    int64_t w_plane;
    int ldw;
    const float* bias;
    const void *down, *up;
    int K, N, rank, n_groups, activation;
    int64_t rows;
    float scale, slope;
    void* y;
    int64_t ldy;
};
template <class T, int RT>
__global__ __launch_bounds__(512) void few_kernel(FewArgs a) {
    constexpr int P = Elem<T>::planes;
    __shared__ float part[8][16][17];
    __shared__ float low[8][16][16 * RT + 1];   // [slice of the depth][row][rank]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16, r = a.rank, K = a.K;
    const int64_t row0 = blockIdx.y * (int64_t)16;
    const int64_t my = min(row0 + l15, a.rows - 1);
    int g = row0 + l15 < a.rows ? a.groups[my] : -1;
    if ((unsigned)g >= (unsigned)a.n_groups) g = -1;
    const T* xr = (const T*)a.x + my * a.ldx;

    f32x4 acc = {0, 0, 0, 0};
    const bf16_t* wr = a.w + (int64_t)(n0 + l15) * a.ldw;
    for (int k0 = 32 * wave; k0 < K; k0 += 256) {
        const int k = k0 + 8 * quad;
        const Planes8<T> xp = to_planes(load8<T>(xr + k, K - k));
        s16x8 wf[P];
#pragma unroll
        for (int p = 0; p < P; ++p) wf[p] = __builtin_bit_cast(s16x8, *reinterpret_cast<const u32x4*>(wr + p * a.w_plane + k));
        acc = mma(wf, xp.p, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][l15][4 * quad + i] = acc[i];

    // u: the waves share the distinct adapters, and with fewer than eight of them the depth too (SL slices of it)
    unsigned pending = (unsigned)__ballot(g >= 0) & 0xffffu;
    int distinct = 0;
    for (unsigned p = pending; p; ++distinct) p &= ~(unsigned)__ballot(g == __builtin_amdgcn_readfirstlane(__shfl(g, __builtin_ctz(p))));
    const int SL = distinct <= 1 ? 8 : distinct <= 2 ? 4 : distinct <= 4 ? 2 : 1, slice = wave % SL;
    for (int at = 0; pending; ++at) {
        const int one = __builtin_amdgcn_readfirstlane(__shfl(g, __builtin_ctz(pending)));
        const unsigned same = (unsigned)__ballot(g == one) & 0xffffu;
        pending &= ~same;
        if (at % (8 / SL) != wave / SL) continue;
        const T* const base = (const T*)a.down + (int64_t)one * r * K;
        f32x4 u[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) u[j] = f32x4{0, 0, 0, 0};
        constexpr int B = RT == 4 ? 2 : 4;   // pieces of the depth whose loads are requested together
        int k0 = 32 * slice;
        for (; k0 + 32 * SL * (B - 1) + 32 <= K; k0 += 32 * SL * B) {
            Raw8<T> xr8[B], ar8[B][RT];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int k = k0 + 32 * SL * b + 8 * quad;
                xr8[b].load(xr + k);
#pragma unroll
                for (int j = 0; j < RT; ++j) ar8[b][j].load(base + (int64_t)min(16 * j + l15, r - 1) * K + k);   // (ranks behind r are not used)
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const Planes8<T> xp = to_planes(xr8[b]);
#pragma unroll
                for (int j = 0; j < RT; ++j) u[j] = mma(to_planes(ar8[b][j]).p, xp.p, u[j]);
            }
        }
        for (; k0 < K; k0 += 32 * SL) {
            const int k = k0 + 8 * quad;
            const Planes8<T> xp = to_planes(load8<T>(xr + k, K - k));
#pragma unroll
            for (int j = 0; j < RT; ++j) u[j] = mma(to_planes(load8<T>(base + (int64_t)min(16 * j + l15, r - 1) * K + k, K - k)).p, xp.p, u[j]);
        }
        if (g == one) {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) low[slice][l15][16 * j + 4 * quad + i] = u[j][i];
        }
    }
    __syncthreads();
    if (SL > 1) {   // the slices' sums, in their order
        for (int i = tid; i < 16 * r; i += 512) {
            const int row = i / r, j = i - row * r;
            float v = low[0][row][j];
            for (int q = 1; q < SL; ++q) v += low[q][row][j];
            low[0][row][j] = v;
        }
        __syncthreads();
    }
    if (tid >= 256) return;
    // thread = (row, column)
    const int row = tid >> 4, col = n0 + (tid & 15);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += part[w][row][tid & 15];
    if (row0 + row >= a.rows || col >= a.N) return;
    const int gr = a.groups[row0 + row];
    if ((unsigned)gr < (unsigned)a.n_groups) {
        const T* b = (const T*)a.up + ((int64_t)gr * a.N + col) * r;
        float s = 0.f;
        for (int j0 = 0; j0 < r; j0 += 8) {
            const Raw8<T> w = load8<T>(b + j0, r - j0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (j0 + e >= r) break;
                s = fmaf(low[0][row][j0 + e], w.get(e), s);
            }
        }
        v = fmaf(s, a.scale, v);
    }
    if (a.bias != nullptr) v += a.bias[col];
    if (a.activation) v = v > 0.f ? v : v * a.slope;
    ((T*)a.y)[(row0 + row) * a.ldy + col] = from_f<T>(v);
}

// =====================================================================================================================
// Gradient of the shared projection from checkpoints:  dW = p^T x  [N][K],  db = sum p  [N]
// Tile 128 x 128, split over the rows; both operands are contracted along their slow dimension: row-major LDS tiles [64 rows][128
// columns] read by the transposing LDS instruction.  x's values are exact in bf16 (one plane), so float32 dy costs three products, not
// six, and bf16 dy one, or two where a slope was applied to it (cut8).  8192 x 512 x 512 bf16: 24 us (two products;
// 19 without an activation) and 5.6 us for the join of 16 parts (eight steps; the rest is the first loads, 64 KB of partial sums a workgroup and
// the launch); 4096 x 1104 x 512 float32: 31 us and 6 us.  256-byte tile rows: the
// 32-byte pieces are XOR-permuted by the row so that the eight rows of half a read differ in their banks.
// =====================================================================================================================
struct WeightGradArgs {
    Source x, mask;
    const void* dy;
    int64_t ldy, rows;
    int N, K, k_tiles, tiles;
    int64_t split_rows;
    float slope;
    float* parts;      // [splits][N * K + N]
};
typedef short tr_v4s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ s16x4 read_tr(const unsigned char* p) {
    return __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr_v4s*)p));
}
__device__ __forceinline__ int tr_swz(int row) { return (row & 3) | ((row >> 1) & 4); }

enum { kNoMask, kMaskElements, kMaskCodes };   // where f' comes from
template <class T> constexpr int grad_planes(int mask) { return sizeof(T) == 4 ? 3 : mask == kNoMask ? 1 : 2; }

// EVEN: N is a multiple of 8.  Which kind of tensor is read is part of the kernel's type: a load behind a branch, even a uniform one,
// made every load in flight be waited for (8192 x 512 x 512, mask of codes: 1.5 us a step of 64 rows instead of 0.6)
template <class T, int MASK, bool EVEN>
__global__ __launch_bounds__(512) void weight_grad_kernel(WeightGradArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    // (in an order that gives the tiles of a split to one XCD, whose L2 they would share: 32768 rows 45 us against 46, 8192 rows 26 against 24)
    const int split = (int)blockIdx.x / a.tiles, tile = (int)blockIdx.x % a.tiles, n0 = (tile / a.k_tiles) * 128, k0 = (tile % a.k_tiles) * 128;
    constexpr int P = grad_planes<T>(MASK), BR = 64, TB = BR * 256;   // smem: [2][P + 1][TB]: planes of p (cut8), then x
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, quad = lane >> 4;
    const int64_t lo = split * a.split_rows, hi = min(lo + a.split_rows, a.rows);
    const int half = wave >> 2, wn = (wave >> 1) & 1, wk = wave & 1;   // waves 0-3 take rows 0-31 of a tile, waves 4-7 rows 32-63

    // pieces of eight columns: thread t has column piece t % 16 of rows t / 16 and t / 16 + 32
    const int pc = tid & 15, pr = tid >> 4;
    // (columns behind the last are read as the last piece: what they add to is not stored)
    const int nc = EVEN ? min(n0 + 8 * pc, a.N - 8) : n0 + 8 * pc, nv = EVEN ? 8 : a.N - nc;
    const int xc = min(k0 + 8 * pc, (int)a.x.ld - 8), mc = MASK == kMaskCodes ? min(n0 + 8 * pc, (int)a.mask.ld - 8) : 0;
    struct Codes { u32x2 code; unsigned exp; };
    struct Ahead { Raw8<T> pw[2], me[2]; Codes mw[2], xw[2]; } ahead[2];   // two tiles on their way
    auto fetch = [&](int64_t row0, Ahead& t) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t at = min(row0 + pr + 32 * q, hi - 1);   // (behind the last row: read again, and set to zero in keep)
            t.pw[q] = load8<T>((const T*)a.dy + at * a.ldy + nc, nv);
            if constexpr (MASK == kMaskElements) t.me[q] = load8<T>((const T*)a.mask.p + at * a.mask.ld + nc, nv);
            if constexpr (MASK == kMaskCodes) read_codes8(a.mask, at, mc, 8, t.mw[q]);
            read_codes8(a.x, at, xc, 8, t.xw[q]);
        }
    };
    const bool sums = k0 == 0;   // these workgroups add up p as well
    float bsum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bsum[e] = 0.f;
    auto keep = [&](unsigned char* buf, int64_t row0, Ahead& t) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int row = pr + 32 * q, at = row * 256 + (((pc >> 1) ^ tr_swz(row)) * 32 + (pc & 1) * 16);
            if (row0 + row >= hi) {
                t.pw[q].zero();
                t.xw[q].code = u32x2{0, 0};
            }
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = t.pw[q].get(e);
                if constexpr (MASK == kMaskCodes) f[e] *= slope_of(t.mw[q].code[e >> 2], e & 3, a.slope);
                if constexpr (MASK == kMaskElements) f[e] = t.me[q].get(e) > 0.f ? f[e] : f[e] * a.slope;
            }
            if (sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) bsum[e] += f[e];
            }
            const Cut8<P> pl = cut8<P, true>(f);   // (x holds no infinities)
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<s16x8*>(buf + p * TB + at) = pl.p[p];
            const float scale = __uint_as_float(t.xw[q].exp << 23);
            const u32x2 x0 = decode4_bf16(t.xw[q].code[0], scale), x1 = decode4_bf16(t.xw[q].code[1], scale);
            *reinterpret_cast<u32x4*>(buf + P * TB + at) = u32x4{x0[0], x0[1], x1[0], x1[1]};
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    // lane's share of a transposed operand: rows 8 quad + l15 / 4 (+ 4) of the wave's 32, columns 4 (l15 % 4) of the 16
    const int fr = 32 * half + 8 * quad + (l15 >> 2);
    auto frag = [&](const unsigned char* buf, int col0) {
        const int piece = (col0 >> 4), off = 8 * (l15 & 3);
        const s16x4 a0 = read_tr(buf + fr * 256 + ((piece ^ tr_swz(fr)) * 32) + off);
        const s16x4 a1 = read_tr(buf + (fr + 4) * 256 + ((piece ^ tr_swz(fr + 4)) * 32) + off);
        return __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto multiply = [&](const unsigned char* buf) {
        s16x8 xf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[j] = frag(buf + P * TB, wk * 64 + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s16x8 pf[P];
#pragma unroll
            for (int p = 0; p < P; ++p) pf[p] = frag(buf + p * TB, wn * 64 + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int p = P - 1; p >= 0; --p) acc[i][j] = mfma32(xf[j], pf[p], acc[i][j]);   // D[k column][n column]
        }
    };
    unsigned char* const buf0 = smem;
    unsigned char* const buf1 = smem + (P + 1) * TB;
    // (rows behind the last one are read as the last and set to zero: every request is in bounds, and no branch is needed)
    if constexpr (sizeof(T) == 2) {
        fetch(lo, ahead[0]);
        fetch(lo + BR, ahead[1]);
        keep(buf0, lo, ahead[0]);
        __syncthreads();
        for (int64_t row0 = lo; row0 < hi; row0 += 2 * BR) {
            fetch(row0 + 2 * BR, ahead[0]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(buf0);
            __builtin_amdgcn_sched_barrier(0);
            keep(buf1, row0 + BR, ahead[1]);
            __syncthreads();
            fetch(row0 + 3 * BR, ahead[1]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(buf1);
            __builtin_amdgcn_sched_barrier(0);
            keep(buf0, row0 + 2 * BR, ahead[0]);
            __syncthreads();
        }
    } else {   // (three planes: the registers of one tile ahead)
        fetch(lo, ahead[0]);
        keep(buf0, lo, ahead[0]);
        __syncthreads();
        unsigned char *now = buf0, *next = buf1;
        for (int64_t row0 = lo; row0 < hi; row0 += BR) {
            fetch(row0 + BR, ahead[0]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(now);
            __builtin_amdgcn_sched_barrier(0);
            keep(next, row0 + BR, ahead[0]);
            __syncthreads();
            unsigned char* const t = now;
            now = next;
            next = t;
        }
    }
    // the two halves' sums
    f32x4* red = reinterpret_cast<f32x4*>(smem);   // [4 waves][16][64]: the tiles are done with (barrier above)
    if (half) {
#pragma unroll
        for (int q = 0; q < 16; ++q) red[((wave & 3) * 16 + q) * 64 + lane] = acc[q / 4][q % 4];
    }
    __syncthreads();
    float* out = a.parts + split * ((int64_t)a.N * a.K + a.N);
    if (!half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + wn * 64 + 16 * i + l15;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = k0 + wk * 64 + 16 * j + 4 * quad;
                const f32x4 v = acc[i][j] + red[(wave * 16 + 4 * i + j) * 64 + lane];
                if (n < a.N && k + 4 <= a.K) {
                    *reinterpret_cast<f32x4_any*>(out + (int64_t)n * a.K + k) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n < a.N && k + e < a.K) out[(int64_t)n * a.K + k + e] = v[e];
                }
            }
        }
    }
    if (sums) {
        __syncthreads();
        float* s = reinterpret_cast<float*>(smem);   // [32 rows][128]
#pragma unroll
        for (int e = 0; e < 8; ++e) s[pr * 128 + 8 * pc + e] = bsum[e];
        __syncthreads();
        if (tid < 128 && n0 + tid < a.N) {
            float v = 0.f;
            for (int i = 0; i < 32; ++i) v += s[i * 128 + tid];
            out[(int64_t)a.N * a.K + n0 + tid] = v;
        }
    }
}
template <class T>
__global__ __launch_bounds__(256) void weight_join_kernel(const float* parts, int splits, int64_t n_weight, int64_t total, T* dw, T* db) {
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (i >= total) return;
    float s = 0.f;
    for (int p = 0; p < splits; ++p) s += parts[p * total + i];
    if (i < n_weight) dw[i] = from_f<T>(s);
    else if (db != nullptr) db[i - n_weight] = from_f<T>(s);
}
// about 256 workgroups, at least 128 rows each
static int64_t weight_splits(int64_t rows, int64_t n, int64_t k, int64_t* split_rows) {
    const int64_t tiles = ceil_div(n, 128) * ceil_div(k, 128);
    int64_t want = tiles < 256 ? 256 / tiles : 1;   // one workgroup a CU
    const int64_t most = ceil_div(rows, 128);
    want = want < most ? want : most;
    *split_rows = round_up(ceil_div(rows, want), 64);
    return ceil_div(rows, *split_rows);
}

// =====================================================================================================================
// Checks that every entry shares
// =====================================================================================================================
static void check_dtype(int dtype) { VH_REQUIRE(dtype == VH_F32 || dtype == VH_BF16, "dtype must be VH_F32 or VH_BF16, not %d", dtype); }
static void check_rows(int64_t rows) { VH_REQUIRE(rows >= 1 && rows <= (int64_t(1) << 30), "rows must be in [1, 2^30], not %lld", (long long)rows); }
static void check_width(int64_t w, const char* what) { VH_REQUIRE(w >= 1 && w <= (1 << 20), "%s must be in [1, 2^20], not %lld", what, (long long)w); }
static void check_groups(int64_t g) { VH_REQUIRE(g >= 1 && g <= kMaxGroups, "the number of groups must be in [1, %d], not %lld", kMaxGroups, (long long)g); }
static void check_rank(int64_t r) { VH_REQUIRE(r >= 1 && r <= kMaxRank, "the rank must be in [1, %d], not %lld", kMaxRank, (long long)r); }
static void check_ptr(const void* p, const char* what) { VH_REQUIRE(p != nullptr, "%s is NULL", what); }
static void check_slope(int activation, float slope) {
    // (below 0 the sign of the value would not tell the derivative)
    VH_REQUIRE(!activation || (slope >= 0.f && slope < __builtin_inff()), "the negative slope must be finite and >= 0");
}
static void check_held(const uint8_t* codes, const uint8_t* exps, const char* what) {
    VH_REQUIRE((codes == nullptr) == (exps == nullptr), "%s: codes and exponents come together", what);
    VH_REQUIRE((uintptr_t)codes % 8 == 0, "%s: codes must be 8-byte aligned", what);
}
static int64_t code_cols(int64_t c) { return round_up(c, kBlockCols); }

static Source source_of(const vh_held* t, int64_t cols, const char* what) {
    check_held(t->codes, t->exponents, what);
    VH_REQUIRE((t->data != nullptr) != (t->codes != nullptr), "%s: either elements or codes", what);
    if (t->codes != nullptr) return {t->codes, t->exponents, code_cols(cols)};
    VH_REQUIRE(t->ld >= cols, "%s: row stride %lld below the %lld columns", what, (long long)t->ld, (long long)cols);
    return {t->data, nullptr, t->ld};
}
static void check_layer(const vh_adapt_layer* l) {
    check_ptr(l, "layer");
    check_dtype(l->dtype);
    check_width(l->n, "n");
    check_width(l->k, "k");
    check_groups(l->groups);
    check_rank(l->rank);
    check_ptr(l->packed, "packed weight");
    VH_REQUIRE((uintptr_t)l->packed % 16 == 0, "packed weight must be 16-byte aligned");
    check_ptr(l->down, "down");
    check_ptr(l->up, "up");
    check_slope(l->activation, l->negative_slope);
    VH_REQUIRE(l->scale == l->scale && fabsf(l->scale) < __builtin_inff(), "scale must be finite");
}
template <class T, int RT>
static void launch_few(const FewArgs& a, hipStream_t s) {
    few_kernel<T, RT><<<dim3((unsigned)ceil_div(a.N, 16), (unsigned)ceil_div(a.rows, 16)), 512, 0, s>>>(a);
    VH_HIP(hipGetLastError());
}
template <class T>
static void few_rank(const FewArgs& a, hipStream_t s) {
    if (a.rank <= 16) launch_few<T, 1>(a, s);
    else if (a.rank <= 32) launch_few<T, 2>(a, s);
    else launch_few<T, 4>(a, s);
}
template <class T, int PP>
static void adapter_first(const AdapterGradArgs& a, hipStream_t s) {
    const int64_t blocks = a.ps.items * ceil_div(a.N, 64) + ceil_div(a.ps.slots * (a.ldp / 8), 1024);
    VH_REQUIRE(fits_a_launch(blocks, 256), "%lld rows of %d columns are too many for one launch", (long long)a.ps.rows, a.N);
    adapter_first_kernel<T, PP><<<(unsigned)blocks, 256, 0, s>>>(a);
    VH_HIP(hipGetLastError());
}
template <class T, int RT, int PP>
static void adapter_grads_rank(const AdapterGradArgs& a, hipStream_t s) {
    const int64_t tiles = ceil_div(a.K, 128) + ceil_div(a.N, 128);
    if constexpr (RT < 4) {
        if (grad_waves(a.ps, a.N, a.K, a.rank) == 4) {
            adapter_grad_kernel<T, RT, 2, 4, PP><<<dim3((unsigned)a.ps.items, (unsigned)tiles), 256, 0, s>>>(a);
            VH_HIP(hipGetLastError());
            return;
        }
    }
    adapter_grad_kernel<T, RT, 2, 1, PP><<<dim3((unsigned)a.ps.items, (unsigned)ceil_div(tiles, 4)), 256, 0, s>>>(a);
    VH_HIP(hipGetLastError());
}
template <class T, int PP>
static void adapter_grads(const AdapterGradArgs& a, hipStream_t s) {
    if (a.rank <= 16) adapter_grads_rank<T, 1, PP>(a, s);
    else if (a.rank <= 32) adapter_grads_rank<T, 2, PP>(a, s);
    else adapter_grads_rank<T, 4, PP>(a, s);
    if (a.ps.rows > a.ps.item_rows) {
        const int64_t multis = a.ps.rows / a.ps.item_rows < a.ps.groups ? a.ps.rows / a.ps.item_rows : a.ps.groups;
        adapter_join_kernel<T><<<dim3((unsigned)ceil_div((int64_t)a.rank * (a.K + a.N), 256), (unsigned)multis), 256, 0, s>>>(a);
        VH_HIP(hipGetLastError());
    }
}
template <class T, int MASK, bool EVEN>
static void launch_weight_grad(const WeightGradArgs& a, int splits, hipStream_t s) {
    const int64_t blocks = (int64_t)a.tiles * splits;
    VH_REQUIRE(fits_a_launch(blocks, 512), "a gradient of %d x %d is too large for one launch", a.N, a.K);
    constexpr int bytes = 2 * (grad_planes<T>(MASK) + 1) * 64 * 256;
    if constexpr (bytes > 65536)
        VH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(weight_grad_kernel<T, MASK, EVEN>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    weight_grad_kernel<T, MASK, EVEN><<<(unsigned)blocks, 512, bytes, s>>>(a);
    VH_HIP(hipGetLastError());
}
template <class T, int MASK>
static void weight_grad_width(const WeightGradArgs& a, int splits, hipStream_t s) {
    if (a.N % 8 == 0) launch_weight_grad<T, MASK, true>(a, splits, s);
    else launch_weight_grad<T, MASK, false>(a, splits, s);
}
template <class T>
static void weight_grad(const WeightGradArgs& a, int splits, void* dweight, void* dbias, hipStream_t s) {
    const int64_t n_weight = (int64_t)a.N * a.K, total = n_weight + a.N;
    VH_REQUIRE(fits_a_launch(ceil_div(total, 256), 256), "a gradient of %d x %d is too large for one launch", a.N, a.K);
    if (a.mask.p == nullptr) weight_grad_width<T, kNoMask>(a, splits, s);
    else if (a.mask.exps == nullptr) weight_grad_width<T, kMaskElements>(a, splits, s);
    else weight_grad_width<T, kMaskCodes>(a, splits, s);
    weight_join_kernel<T><<<(unsigned)ceil_div(total, 256), 256, 0, s>>>(a.parts, splits, n_weight, total, (T*)dweight, (T*)dbias);
    VH_HIP(hipGetLastError());
}
// the backward pass's scratch, in words: v, up turned around, p, the parts of groups of several items
struct BackwardScratch {
    int64_t ldp, turned, p, parts, words;
};
static BackwardScratch backward_scratch(const PlanShape& ps, int64_t n, int64_t k, int64_t rank, int dtype) {
    BackwardScratch b{};
    const int64_t es = dtype == VH_BF16 ? 2 : 4, planes = dtype == VH_BF16 ? 2 : 3;   // (bf16 without an activation: one, of two)
    b.ldp = round_up(n, 8);
    b.turned = round_up(ps.rows * rank, 4);
    b.p = b.turned + round_up(ps.groups * rank * b.ldp * es / 4, 4);
    b.parts = b.p + round_up(planes * ps.slots * b.ldp / 2, 4);
    b.words = b.parts + (ps.rows > ps.item_rows ? 2 * (ps.rows / ps.item_rows) * rank * (n + k) : 0);
    return b;
}

}  // namespace adapt
}  // namespace vh

using namespace vh;
using namespace vh::adapt;

extern "C" {

int vh_rows_plan_size(int64_t rows, int64_t groups, int64_t* plan_words, int64_t* scratch_words) {
    return guarded([&] {
        check_rows(rows);
        check_groups(groups);
        check_ptr(plan_words, "plan_words");
        check_ptr(scratch_words, "scratch_words");
        *plan_words = plan_shape(rows, groups).words;
        *scratch_words = plan_is_small(rows, groups) ? 0 : (groups + 1) * (plan_pieces(rows) + 1);
    });
}

int vh_rows_plan(const int32_t* row_groups, int64_t rows, int64_t groups, int32_t* plan, int32_t* scratch, void* stream) {
    return guarded([&] {
        check_rows(rows);
        check_groups(groups);
        check_ptr(row_groups, "row_groups");
        check_ptr(plan, "plan");
        VH_REQUIRE((uintptr_t)plan % 16 == 0, "plan must be 16-byte aligned");
        const PlanShape ps = plan_shape(rows, groups);
        hipStream_t s = (hipStream_t)stream;
        int bits = 1;
        while ((1 << bits) < groups + 2) ++bits;   // keys 0 .. groups + 1
        if (plan_is_small(rows, groups)) {
            plan_small_kernel<<<(unsigned)ceil_div(rows, 1024), 1024, 18 * (groups + 1) * sizeof(int), s>>>(row_groups, plan, ps, bits);
            VH_HIP(hipGetLastError());
            return;
        }
        check_ptr(scratch, "scratch");
        const int pieces = (int)plan_pieces(rows);
        const int64_t seg = round_up(ceil_div(rows, pieces), 64);
        const size_t lds = (groups + 1) * sizeof(int);
        int* totals = scratch + (groups + 1) * pieces;
        if (lds > 65536) {
            VH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(plan_count_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
            VH_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(plan_place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        }
        plan_count_kernel<<<pieces, 64, lds, s>>>(row_groups, scratch, ps, seg, pieces);
        VH_HIP(hipGetLastError());
        plan_scan_kernel<<<(unsigned)(groups + 1), 64, 0, s>>>(scratch, (int)groups, pieces);
        VH_HIP(hipGetLastError());
        plan_offsets_kernel<<<1, 1024, 0, s>>>(plan, totals, ps);
        VH_HIP(hipGetLastError());
        plan_place_kernel<<<pieces, 64, lds, s>>>(row_groups, scratch, plan, ps, seg, pieces, bits);
        VH_HIP(hipGetLastError());
    });
}

int vh_adapt_weight_size(int64_t n, int64_t k, int dtype, int64_t* bytes) {
    return guarded([&] {
        check_dtype(dtype);
        check_width(n, "n");
        check_width(k, "k");
        check_ptr(bytes, "bytes");
        *bytes = weight_shape(n, k, dtype).bytes;
    });
}

int vh_adapt_weight_pack(const void* weight, int64_t ld, const void* bias, int64_t n, int64_t k, int dtype, void* packed, void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        check_width(n, "n");
        check_width(k, "k");
        check_ptr(weight, "weight");
        check_ptr(packed, "packed");
        VH_REQUIRE(ld >= k, "row stride %lld below the %lld columns", (long long)ld, (long long)k);
        VH_REQUIRE((uintptr_t)packed % 16 == 0, "packed weight must be 16-byte aligned");
        const WeightShape ws = weight_shape(n, k, dtype);
        float* out_bias = reinterpret_cast<float*>((char*)packed + ws.bias_off);
        VH_REQUIRE(fits_a_launch(ceil_div(ws.fwd + ws.bwd, 256), 256), "a weight of %lld x %lld is too large for one launch", (long long)n, (long long)k);
        const unsigned blocks = (unsigned)ceil_div(ws.fwd + ws.bwd, 256);
        if (dtype == VH_BF16)
            pack_weight_kernel<bf16_t><<<blocks, 256, 0, (hipStream_t)stream>>>((const bf16_t*)weight, ld, (const bf16_t*)bias, (int)n, (int)k,
                                                                                (bf16_t*)packed, out_bias, ws);
        else
            pack_weight_kernel<float><<<blocks, 256, 0, (hipStream_t)stream>>>((const float*)weight, ld, (const float*)bias, (int)n, (int)k,
                                                                               (bf16_t*)packed, out_bias, ws);
        VH_HIP(hipGetLastError());
    });
}

int vh_adapt_forward(const vh_adapt_layer* l, const void* x, int64_t ldx, int64_t rows, const int32_t* plan, void* y, int64_t ldy, float* low,
                     uint8_t* codes, uint8_t* exponents, void* stream) {
    return guarded([&] {
        check_layer(l);
        check_rows(rows);
        check_ptr(x, "x");
        check_ptr(y, "y");
        check_ptr(plan, "plan");
        VH_REQUIRE(ldx >= l->k && ldy >= l->n, "row strides below the number of columns");
        check_held(codes, exponents, "checkpoint of y");
        VH_REQUIRE((uintptr_t)low % 16 == 0, "low must be 16-byte aligned");
        const WeightShape ws = weight_shape(l->n, l->k, l->dtype);
        const int es = l->dtype == VH_BF16 ? 2 : 4;
        LinArgs a{};
        a.x = x;
        a.ldx = ldx;
        a.slope = l->negative_slope;
        a.activation = l->activation;
        a.w = (const bf16_t*)l->packed;
        a.w_plane = ws.fwd;
        a.ldw = (int)ws.kq;
        a.bias = reinterpret_cast<const float*>((const char*)l->packed + ws.bias_off);
        a.inner = l->down;
        a.ld_inner = l->k;
        a.outer = l->up;
        a.K = (int)l->k;
        a.N = (int)l->n;
        a.rank = (int)l->rank;
        a.scale = l->scale;
        a.low_scale = 1.f;
        a.low = low;
        a.y = y;
        a.ldy = ldy;
        a.codes = codes;
        a.ldc = code_cols(l->n);
        a.exps = exponents;
        a.plan = plan;
        a.ps = plan_shape(rows, l->groups);
        const int64_t x_bytes = ((rows - 1) * ldx + l->k) * es;
        a.dma = es == 2 && l->k % 8 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && x_bytes < 0xfffffff0ll;   // (down is read at any alignment)
        a.x_bytes = a.dma ? (unsigned)x_bytes : 0;
        if (l->dtype == VH_BF16) launch_linear_bf16(a, false, (hipStream_t)stream);
        else launch_linear_f32(a, false, (hipStream_t)stream);
    });
}

int vh_adapt_forward_few(const vh_adapt_layer* l, const void* x, int64_t ldx, int64_t rows, const int32_t* row_groups, void* y, int64_t ldy, void* stream) {
    return guarded([&] {
        check_layer(l);
        check_rows(rows);
        check_ptr(x, "x");
        check_ptr(y, "y");
        check_ptr(row_groups, "row_groups");
        VH_REQUIRE(rows <= 65535 * 16, "too many rows for this entry");
        VH_REQUIRE(ldx >= l->k && ldy >= l->n, "row strides below the number of columns");
        const WeightShape ws = weight_shape(l->n, l->k, l->dtype);
        FewArgs a{};
        a.x = x;
        a.ldx = ldx;
        a.groups = row_groups;
        a.w = (const bf16_t*)l->packed;
        a.w_plane = ws.fwd;
        a.ldw = (int)ws.kq;
        a.bias = reinterpret_cast<const float*>((const char*)l->packed + ws.bias_off);
        a.down = l->down;
        a.up = l->up;
        a.K = (int)l->k;
        a.N = (int)l->n;
        a.rank = (int)l->rank;
        a.n_groups = (int)l->groups;
        a.activation = l->activation;
        a.rows = rows;
        a.scale = l->scale;
        a.slope = l->negative_slope;
        a.y = y;
        a.ldy = ldy;
        if (l->dtype == VH_BF16) few_rank<bf16_t>(a, (hipStream_t)stream);
        else few_rank<float>(a, (hipStream_t)stream);
    });
}

int vh_adapt_backward_size(int64_t rows, int64_t groups, int64_t n, int64_t k, int64_t rank, int dtype, int64_t* scratch_words) {
    return guarded([&] {
        check_rows(rows);
        check_groups(groups);
        check_width(n, "n");
        check_width(k, "k");
        check_rank(rank);
        check_ptr(scratch_words, "scratch_words");
        check_dtype(dtype);
        *scratch_words = backward_scratch(plan_shape(rows, groups), n, k, rank, dtype).words;
    });
}

int vh_adapt_backward(const vh_adapt_layer* l, const void* dy, int64_t lddy, const vh_held* x, const vh_held* y, const float* low, int64_t rows,
                      const int32_t* plan, void* dx, int64_t lddx, void* ddown, void* dup, float* scratch, void* stream) {
    return guarded([&] {
        check_layer(l);
        check_rows(rows);
        check_ptr(dy, "dy");
        check_ptr(x, "x");
        check_ptr(low, "low");
        check_ptr(plan, "plan");
        check_ptr(ddown, "ddown");
        check_ptr(dup, "dup");
        check_ptr(scratch, "scratch");
        VH_REQUIRE(lddy >= l->n && (dx == nullptr || lddx >= l->k), "row strides below the number of columns");
        VH_REQUIRE(!l->activation || y != nullptr, "the layer's output is needed for the derivative of its activation");
        const Source xs = source_of(x, l->k, "x");
        Source mask = {nullptr, nullptr, 0};
        if (l->activation) mask = source_of(y, l->n, "y");
        const PlanShape ps = plan_shape(rows, l->groups);
        VH_REQUIRE((uintptr_t)scratch % 16 == 0, "scratch must be 16-byte aligned");
        hipStream_t s = (hipStream_t)stream;
        AdapterGradArgs g{};
        g.x = xs;
        g.mask = mask;
        g.dy = dy;
        g.ldy = lddy;
        g.low = low;
        g.v = scratch;
        g.ddown = ddown;
        g.dup = dup;
        g.up = l->up;
        const BackwardScratch bs = backward_scratch(ps, l->n, l->k, l->rank, l->dtype);
        g.turned = scratch + bs.turned;
        g.p = reinterpret_cast<bf16_t*>(scratch + bs.p);
        g.ldp = bs.ldp;
        g.parts = scratch + bs.parts;
        g.K = (int)l->k;
        g.N = (int)l->n;
        g.rank = (int)l->rank;
        g.scale = l->scale;
        g.slope = l->negative_slope;
        g.plan = plan;
        g.ps = ps;
        const WeightShape ws = weight_shape(l->n, l->k, l->dtype);
        LinArgs a{};
        a.x = g.p;
        a.ldx = bs.ldp;
        a.w = (const bf16_t*)l->packed + ws.planes * ws.fwd;
        a.w_plane = ws.bwd;
        a.ldw = (int)ws.nq;
        a.inner = g.turned;
        a.ld_inner = bs.ldp;
        a.outer = l->down;
        a.K = (int)l->n;
        a.N = (int)l->k;
        a.rank = (int)l->rank;
        a.scale = a.low_scale = l->scale;
        a.low = scratch;   // v
        a.y = dx;
        a.ldy = lddx;
        a.plan = plan;
        a.ps = ps;
        if (l->dtype == VH_F32) {
            a.x_planes = 3;
            adapter_first<float, 3>(g, s);
            launch_linear_f32(a, true, s);
            adapter_grads<float, 3>(g, s);
        } else if (mask.p != nullptr) {
            a.x_planes = 2;
            adapter_first<bf16_t, 2>(g, s);
            launch_linear_bf16(a, true, s);
            adapter_grads<bf16_t, 2>(g, s);
        } else {
            a.x_planes = 1;
            adapter_first<bf16_t, 1>(g, s);
            launch_linear_bf16(a, true, s);
            adapter_grads<bf16_t, 1>(g, s);
        }
    });
}

int vh_debug_adapt_choice(int64_t rows, int64_t groups, int64_t n, int64_t k, int64_t rank, int dtype, int* forward_tile, int* backward_tile, int* waves) {
    return guarded([&] {
        check_rows(rows);
        check_groups(groups);
        check_width(n, "n");
        check_width(k, "k");
        check_rank(rank);
        check_dtype(dtype);
        check_ptr(forward_tile, "forward_tile");
        check_ptr(backward_tile, "backward_tile");
        check_ptr(waves, "waves");
        const PlanShape ps = plan_shape(rows, groups);
        *forward_tile = linear_tile(ps.subs, n, dtype == VH_F32);
        *backward_tile = linear_tile(ps.subs, k, dtype == VH_F32);
        *waves = grad_waves(ps, n, k, rank);
    });
}

int vh_debug_adapt_item_reads(int64_t rows, int64_t groups, int32_t first, int32_t count, int64_t* highest, int64_t* slots) {
    return guarded([&] {
        check_rows(rows);
        check_groups(groups);
        check_ptr(highest, "highest");
        check_ptr(slots, "slots");
        *slots = plan_shape(rows, groups).slots;
        *highest = -1;
        for (int i = 0; i < (count > 32 ? count : 32); ++i) {   // (up to 32 rows a step, the first of them asked for whatever the count)
            const int64_t at = item_slot(first, count, i, *slots);
            if (at > *highest) *highest = at;
        }
    });
}

int vh_checkpoint8(const void* x, int64_t ld, int64_t rows, int64_t cols, int dtype, uint8_t* codes, uint8_t* exponents, void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        check_rows(rows);
        check_width(cols, "cols");
        check_ptr(x, "x");
        check_ptr(codes, "codes");
        check_held(codes, exponents, "checkpoint");
        VH_REQUIRE(ld >= cols, "row stride %lld below the %lld columns", (long long)ld, (long long)cols);
        const int64_t blocks = ceil_div(rows * (code_cols(cols) / 8), 256);
        const unsigned grid = (unsigned)(blocks < 8192 ? blocks : 8192);
        if (dtype == VH_BF16) checkpoint_kernel<bf16_t><<<grid, 256, 0, (hipStream_t)stream>>>((const bf16_t*)x, ld, rows, (int)cols, codes, exponents);
        else checkpoint_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>((const float*)x, ld, rows, (int)cols, codes, exponents);
        VH_HIP(hipGetLastError());
    });
}

int vh_checkpoint8_restore(const uint8_t* codes, const uint8_t* exponents, int64_t rows, int64_t cols, int dtype, void* out, void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        check_rows(rows);
        check_width(cols, "cols");
        check_ptr(codes, "codes");
        check_ptr(out, "out");
        check_held(codes, exponents, "checkpoint");
        const int64_t blocks = ceil_div(rows * (code_cols(cols) / 8), 256);
        const unsigned grid = (unsigned)(blocks < 8192 ? blocks : 8192);
        if (dtype == VH_BF16) restore_kernel<bf16_t><<<grid, 256, 0, (hipStream_t)stream>>>(codes, exponents, rows, (int)cols, (bf16_t*)out);
        else restore_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(codes, exponents, rows, (int)cols, (float*)out);
        VH_HIP(hipGetLastError());
    });
}

int vh_checkpoint8_weight_grad_size(int64_t rows, int64_t n, int64_t k, int64_t* scratch_words) {
    return guarded([&] {
        check_rows(rows);
        check_width(n, "n");
        check_width(k, "k");
        check_ptr(scratch_words, "scratch_words");
        int64_t split_rows;
        *scratch_words = weight_splits(rows, n, k, &split_rows) * (n * k + n);
    });
}

int vh_checkpoint8_weight_grad(const void* dy, int64_t lddy, const vh_held* x, const vh_held* y, float negative_slope, int64_t rows, int64_t n, int64_t k,
                               int dtype, void* dweight, void* dbias, float* scratch, void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        check_rows(rows);
        check_width(n, "n");
        check_width(k, "k");
        check_ptr(dy, "dy");
        check_ptr(x, "x");
        check_ptr(dweight, "dweight");
        check_ptr(scratch, "scratch");
        VH_REQUIRE(lddy >= n, "row stride %lld below the %lld columns", (long long)lddy, (long long)n);
        check_slope(y != nullptr, negative_slope);
        WeightGradArgs a{};
        a.x = source_of(x, k, "x");
        VH_REQUIRE(a.x.exps != nullptr, "x must be a checkpoint");
        if (y != nullptr) a.mask = source_of(y, n, "y");
        a.dy = dy;
        a.ldy = lddy;
        a.rows = rows;
        a.N = (int)n;
        a.K = (int)k;
        a.k_tiles = (int)ceil_div(k, 128);
        a.slope = negative_slope;
        a.parts = scratch;
        const int64_t splits = weight_splits(rows, n, k, &a.split_rows);
        const int64_t tiles = ceil_div(n, 128) * a.k_tiles;
        a.tiles = (int)tiles;
        if (dtype == VH_BF16) weight_grad<bf16_t>(a, (int)splits, dweight, dbias, (hipStream_t)stream);
        else weight_grad<float>(a, (int)splits, dweight, dbias, (hipStream_t)stream);
    });
}

}  // extern "C"
