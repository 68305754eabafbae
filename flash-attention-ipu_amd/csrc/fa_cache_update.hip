// What changes the state of a block cache: block tables and slots of a step, and new keys and values as e4m3 codes.
#include <hip/hip_runtime.h>

#include "fa_cache.h"
#include "fa_params.h"

namespace fa {
namespace {

// ---- block tables, positions, slots ------------------------------------------------------------------------------------------------------
// Requests b = 0 .. B-1 hold held[b] tokens in ceil(held / P) blocks; n[b] tokens come (n < 0: the request ends).
//   1. the blocks of the requests that end are put behind the free ones, in the order of the requests and of their blocks;
//   2. cu = running sum of max(n, 0); a request fits if cu[b+1] <= T and its blocks fit the table; its need is the number of blocks to add;
//      it is served if it fits and needs nothing or the needs of all that fit up to and including it are there;
//   3. blocks are taken from the end of the free list, in the order of the requests; positions and slots follow.
// Bound: latency - a few kilobytes through one workgroup, three scans (64 requests of a token: 4.9 us; 512 of up to 257 tokens, 16 of them ending: 11.5 us, and 3.8 for the
// slots).  Sums saturate at 2^31 - 1 (which stays associative, so that the
// scan order does not matter) where lengths add up to more.
constexpr int kScanThreads = 1024;
constexpr int kBatch = 4;       // entries per thread whose loads are in flight together

__device__ __forceinline__ int sat_add(int a, int b) {
    const unsigned s = (unsigned)a + (unsigned)b;
    return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}
// inclusive scan with saturation over a wave, through the data-parallel moves: inside rows of 16 lanes, then the rows' last lanes onto the rows behind them
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int x) {
    return sat_add(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_scan(int x) {
    x = scan_step<0x111, 0xf>(x);      // row_shr 1, 2, 4, 8
    x = scan_step<0x112, 0xf>(x);
    x = scan_step<0x114, 0xf>(x);
    x = scan_step<0x118, 0xf>(x);
    x = scan_step<0x142, 0xa>(x);      // row_bcast 15 onto rows 1 and 3
    return scan_step<0x143, 0xc>(x);   // row_bcast 31 onto rows 2 and 3
}
// exclusive scans of N numbers over the workgroup; totals are every thread's
template <int N>
__device__ __forceinline__ void block_scan(const int (&x)[N], int (&before)[N], int (&total)[N], int (*waves)[kScanThreads / 64]) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int incl = wave_scan(x[n]);
        if (lane == 63) waves[n][wave] = incl;
        const int prev = __builtin_amdgcn_update_dpp(0, incl, 0x138, 0xf, 0xf, false);      // wave_shr 1
        before[n] = lane ? prev : 0;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        // the waves' sums, scanned by every wave for itself
        const int sums = wave_scan(lane < kScanThreads / 64 ? waves[n][lane] : 0);
        total[n] = __builtin_amdgcn_readlane(sums, kScanThreads / 64 - 1);
        const int ahead = __builtin_amdgcn_readlane(sums, wave ? __builtin_amdgcn_readfirstlane(wave) - 1 : 0);
        before[n] = sat_add(wave ? ahead : 0, before[n]);
    }
    __syncthreads();
}
// largest i in [0, n) with first[i] <= x; first is ascending, first[0] <= x
__device__ __forceinline__ int find(const int* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ int blocks_of(int64_t tokens, int shift) { return (int)((tokens + (1 << shift) - 1) >> shift); }

// position and slot of token t of request b, which starts at `start` and has `granted` of its tokens granted (all or none) and `total` held then
__device__ __forceinline__ void place(const TablesParams& p, int t, int b, int start, int granted, int total) {
    int pos = -1, slot = -1;
    if (granted > 0) {
        pos = total - granted + (t - start);
        const int block = p.tables[(int64_t)b * p.table_stride + (pos >> p.shift)];
        if (block >= 0) slot = (block << p.shift) + (pos & ((1 << p.shift) - 1));
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
}

__global__ __launch_bounds__(kScanThreads) void cache_tables_kernel(TablesParams p) {
    __shared__ int waves[1][kScanThreads / 64], first[kScanThreads], start[kScanThreads], have_s[kScanThreads], served_to;
    const int tid = (int)threadIdx.x;
    int free = *p.free_in;
    free = free < 0 ? 0 : free > p.pool_size ? p.pool_size : free;
    // 1. ended requests' blocks
    for (int base = 0; base < p.B; base += kScanThreads) {
        const int b = base + tid;
        const bool ends = b < p.B && p.new_lens[b] < 0;
        if (!__syncthreads_or(ends)) continue;
        const int held = ends ? max(p.seq_in[b], 0) : 0;
        const int back[1] = {ends ? min(blocks_of(held, p.shift), p.width) : 0};
        int at[1], total[1];
        block_scan<1>(back, at, total, waves);
        first[tid] = at[0];
        __syncthreads();
        const int bound = min(total[0], p.pool_size - free);
        for (int i0 = tid; i0 < bound; i0 += kBatch * kScanThreads) {
            int id[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * kScanThreads;
                if (i >= bound) continue;
                const int r = find(first, min(p.B - base, kScanThreads), i);
                id[k] = p.tables[(int64_t)(base + r) * p.table_stride + (i - first[r])];
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                if (i0 + k * kScanThreads < bound) p.pool[free + i0 + k * kScanThreads] = id[k];
        }
        __syncthreads();
        free = min(sat_add(free, total[0]), p.pool_size);
    }
    // 2. and 3.
    int tokens = 0, needed = 0, taken = 0;     // running sums over the chunks of requests
    for (int base = 0; base < p.B; base += kScanThreads) {
        const int b = base + tid, here = min(p.B - base, kScanThreads);
        const bool in = b < p.B;
        const int n = in ? p.new_lens[b] : 0, count = max(n, 0), held = in ? max(p.seq_in[b], 0) : 0;
        const int have = blocks_of(held, p.shift);
        const int64_t after = ((int64_t)held + count + (1 << p.shift) - 1) >> p.shift;
        int my_start, my_end, need, before;
        bool fits = in && n >= 0 && after <= p.width;
        {
            const int x[1] = {count};
            int y[1], total[1];
            block_scan<1>(x, y, total, waves);
            my_start = sat_add(tokens, y[0]);
            my_end = sat_add(my_start, count);
            tokens = sat_add(tokens, total[0]);
            fits = fits && my_end <= p.T;
        }
        {
            need = fits ? (int)after - have : 0;
            const int x[1] = {need};
            int y[1], total[1];
            if (tid == 0) served_to = taken;
            block_scan<1>(x, y, total, waves);
            before = sat_add(needed, y[0]);
            needed = sat_add(needed, total[0]);
        }
        // (needs add up: once one is not met, none behind it is, so that a served request's blocks begin at `before`)
        const bool served = fits && (need == 0 || sat_add(before, need) <= free);
        const int granted = served ? count : 0;
        if (served && need > 0) atomicMax(&served_to, before + need);
        first[tid] = before;
        have_s[tid] = have;
        __syncthreads();
        const int upto = served_to;
        for (int k0 = taken + tid; k0 < upto; k0 += kBatch * kScanThreads) {
            int id[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) id[i] = k0 + i * kScanThreads < upto ? p.pool[free - 1 - k0 - i * kScanThreads] : 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int k = k0 + i * kScanThreads;
                if (k >= upto) continue;
                const int r = find(first, here, k);
                p.tables[(int64_t)(base + r) * p.table_stride + have_s[r] + (k - first[r])] = id[i];
            }
        }
        taken = upto;
        const int held_after = n < 0 ? 0 : held + granted;
        if (in) {
            p.seq_out[b] = held_after;
            p.granted[b] = granted;
            p.cu_new[b] = my_start;
            if (b == p.B - 1) p.cu_new[p.B] = my_end;
        }
        __syncthreads();
        if (p.fused) {
            // the tokens of this chunk of requests; first / start / have_s serve as request starts, grants and lengths
            first[tid] = my_start;
            start[tid] = granted;
            have_s[tid] = held_after;
            __syncthreads();
            const int from = base == 0 ? 0 : first[0], to = min(tokens, p.T);
            for (int t = from + tid; t < to; t += kScanThreads) {
                const int r = find(first, here, t);
                place(p, t, base + r, first[r], start[r], have_s[r]);
            }
            __syncthreads();
        }
    }
    if (p.fused)
        for (int t = min(tokens, p.T) + tid; t < p.T; t += kScanThreads) p.positions[t] = p.slots[t] = -1;
    if (tid == 0) *p.free_out = free - taken;
}

constexpr int kSlotThreads = 256, kSlotStage = 2048;
__global__ __launch_bounds__(kSlotThreads) void cache_slots_kernel(TablesParams p) {
    __shared__ int staged[kSlotStage];
    const int t = (int)blockIdx.x * kSlotThreads + (int)threadIdx.x;
    const int* first = p.cu_new;
    if (p.B <= kSlotStage) {                   // (B + 1 entries; the last one bounds the tokens and is read from memory)
        for (int i = (int)threadIdx.x; i < p.B; i += kSlotThreads) staged[i] = p.cu_new[i];
        __syncthreads();
        first = staged;
    }
    if (t >= p.T) return;
    if (t >= p.cu_new[p.B]) {
        p.positions[t] = p.slots[t] = -1;
        return;
    }
    const int b = find(first, p.B, t);
    place(p, t, b, first[b], p.granted[b], p.seq_out[b]);
}

// ---- new keys and values -----------------------------------------------------------------------------------------------------------------
// A run is a stretch of tokens whose slots follow each other inside one block.  For a run, a head and one of the two caches:
//   A = largest finite |x|;  wanted = 2^e, the smallest power of two with A <= 448 * 2^e (e >= -100);
//   a run that begins its block sets the scale to `wanted`; any other run raises it to max(scale, wanted), and where that changes it every
//   code of the block is brought to the new scale;  codes = nearest e4m3 of x / scale (ties to even); inf and NaN become the code of NaN.
// Scales are powers of two because codes carry their own exponent: x / scale is exact, growing a scale only moves the codes' exponents (exact
// but for what falls under the smallest code), and nothing is gained by filling the last fraction of the top binade.
// Bound: memory (2 bytes in, 1 byte out per value) for prompts (24 of up to 2048 tokens, 8 heads of 128: 29.7 us = 5.1 TB/s from the caches, 37.7 us = 4.0 from memory),
// latency for a step (64 tokens: 6.0 us).  A workgroup owns `window` tokens of one head and cache;
// the runs that begin in them are its work - a run is never shared, so scales need no atomics.  One or two long runs are taken by the whole workgroup,
// others by a wave each.
// A work item is eight columns of four consecutive tokens: 16-byte loads, the values stay in registers between the maximum and the codes, and
// both layouts store whole words - eight bytes of a key row, or (columns down the lanes) four tokens of a value column.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Bits;
template <> struct Bits<_Float16> {
    static constexpr unsigned top = 0x7c00u;
    typedef _Float16 vec2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float f(unsigned u) { return (float)__builtin_bit_cast(_Float16, (unsigned short)u); }
    // four finite values / 2^e -> four codes, one rounding: the instruction divides by the scale's power of two before it rounds
    static __device__ __forceinline__ unsigned codes(unsigned a, unsigned b, float scale) {
        s16x2 r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(vec2, a), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(vec2, b), scale, true);
        return __builtin_bit_cast(unsigned, r);
    }
};
template <> struct Bits<__bf16> {
    static constexpr unsigned top = 0x7f80u;
    typedef __bf16 vec2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float f(unsigned u) { return __builtin_bit_cast(float, u << 16); }
    static __device__ __forceinline__ unsigned codes(unsigned a, unsigned b, float scale) {
        s16x2 r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(vec2, a), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(vec2, b), scale, true);
        return __builtin_bit_cast(unsigned, r);
    }
};

// |x| <= 448 by the choice of the scale, except inf and NaN, which become the code of NaN
__device__ __forceinline__ unsigned codes2(float a, float b) {
    const float inf = __builtin_inff();
    a = __builtin_fabsf(a) == inf ? __builtin_nanf("") : a;
    b = __builtin_fabsf(b) == inf ? __builtin_nanf("") : b;
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
__device__ __forceinline__ unsigned rescale4(unsigned w, float f) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return codes2(lo[0] * f, lo[1] * f) | codes2(hi[0] * f, hi[1] * f) << 16;
}
__device__ __forceinline__ float wanted_scale(float largest) {
    const unsigned u = __builtin_bit_cast(unsigned, largest);
    int e = (int)(u >> 23) - 126 - 9 + ((u & 0x7fffffu) > 0x600000u);    // largest = m 2^E, m in [0.5, 1): e = E - 9 + (m > 0.875)
    e = e < -100 ? -100 : e;
    return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}
__device__ __forceinline__ unsigned wave_max(unsigned x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned y = (unsigned)__shfl_xor((int)x, d);
        x = x > y ? x : y;
    }
    return x;
}
// bytes of four rows of four -> four columns of four
__device__ __forceinline__ void transpose4(unsigned (&r)[4]) {
    const unsigned a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
    const unsigned c = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
    r[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    r[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    r[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    r[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// One run: tokens t0 .. t0 + n - 1 into positions off .. off + n - 1 of a block.  NT = 64 (a wave) or 256 (the workgroup).
// HOLD: items per thread that stay in registers between the maximum and the codes: one where a whole block is one item per thread of a workgroup
// (24 prompts of up to 2048, blocks of 64, 8 heads of 128: 30.4 us, with two 32.0; 16384 tokens, heads of 64: 17.0 and 18.8), else two (16384 tokens, blocks of 128:
// 26.3 us, with one 28.9).
template <typename T, int W, int HOLD, bool KEYS, int NT>
__device__ __forceinline__ void append_run(const AppendParams& p, int t0, int n, int64_t block, int off, int head, unsigned* shared_max) {
    constexpr int S = KEYS ? 0 : 1, WC = W / 8;                           // column chunks of a row
    const int tid = (int)threadIdx.x & (NT - 1);
    const int P = 1 << p.shift, chunks = p.D >> 3;
    const int g0 = off >> 2, groups = ((off + n + 3) >> 2) - g0;          // groups of four positions that the run touches
    // keys: neighbouring lanes take a row's chunks; values: neighbouring lanes take up to sixteen groups of one chunk (a 64-byte piece of every column)
    const int lg = groups > 4 ? 4 : groups > 1 ? 2 : 0;
    const int items = KEYS ? groups * WC : (((groups - 1) >> lg) + 1) * (WC << lg);
    const int64_t st = p.x_st[S];
    const T* x = (const T*)p.x[S] + (int64_t)head * p.x_sh[S] + (int64_t)t0 * st;
    uint8_t* tile = (uint8_t*)p.cache[S] + block * p.block_stride[S] + (int64_t)head * P * W;
    float* scale = p.scale[S] + block * p.scale_stride[S] + head;
    float old = off ? *scale : 0.f;

    const auto place = [&](int i, int& g, int& c) {                       // item i: position group g, column chunk c
        if (KEYS) { g = g0 + i / WC; c = i % WC; }
        else { const int hi = i >> lg; g = g0 + ((hi / WC) << lg) + (i & ((1 << lg) - 1)); c = hi % WC; }
    };
    const auto load = [&](int i, u32x4v (&v)[4]) {
        int g, c;
        place(i, g, c);
        const int k0 = 4 * g - off;                                       // run index of the group's first position
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (k0 + r >= 0 && k0 + r < n && c < chunks) v[r] = *(const u32x4v*)(x + (int64_t)(k0 + r) * st + 8 * c);
            else v[r] = u32x4v{0, 0, 0, 0};
        }
    };
    const auto look = [&](const u32x4v (&v)[4], u16x2 m) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int q = 0; q < 4; ++q) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[r][q] & 0x7fff7fffu));
        return m;
    };
    const auto look_finite = [&](const u32x4v (&v)[4], u16x2 m) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const unsigned lo = v[r][q] & 0x7fffu, hi = (v[r][q] >> 16) & 0x7fffu;
                m[0] = lo < Bits<T>::top && lo > m[0] ? lo : m[0];
                m[1] = hi < Bits<T>::top && hi > m[1] ? hi : m[1];
            }
        return m;
    };
    u32x4v held[HOLD][4];
    const auto over_all = [&](auto f) {
        u16x2 m = {0, 0};
#pragma unroll
        for (int h = 0; h < HOLD; ++h)
            if (tid + h * NT < items) m = f(held[h], m);
        for (int i = tid + HOLD * NT; i < items; i += NT) {
            u32x4v v[4];
            load(i, v);
            m = f(v, m);
        }
        unsigned largest = wave_max(m[0] > m[1] ? m[0] : m[1]);
        if constexpr (NT == 256) {
            if ((threadIdx.x & 63) == 0) shared_max[threadIdx.x >> 6] = largest;
            __syncthreads();
            largest = max(max(shared_max[0], shared_max[1]), max(shared_max[2], shared_max[3]));
            __syncthreads();
        }
        return (unsigned)__builtin_amdgcn_readfirstlane((int)largest);
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (tid + h * NT < items) load(tid + h * NT, held[h]);
    asm volatile("" : "+v"(old));             // (here, before the maximum's barrier: the first thread stores the scale behind it)
    unsigned largest = over_all(look);
    const bool finite = largest < Bits<T>::top;
    if (!finite) largest = over_all(look_finite);
    const float wanted = wanted_scale(Bits<T>::f(largest));
    const float now = off == 0 ? wanted : old > wanted ? old : wanted;
    if (off != 0 && now != old) {              // (uniform over the NT threads)
        const float f = old / now;
        for (int i = tid; i < P * W / 16; i += NT) {
            u32x4v w = *(const u32x4v*)(tile + 16 * i);
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = rescale4(w[q], f);
            *(u32x4v*)(tile + 16 * i) = w;
        }
        __threadfence();                       // these stores are done before the run's own bytes are written
        if constexpr (NT == 256) __syncthreads();
    }
    if (tid == 0) *scale = now;
    // a power of two that the conversion takes, and nothing but finite values
    const unsigned nb = __builtin_bit_cast(unsigned, now);
    const bool fast = finite && (nb & 0x807fffffu) == 0u && nb != 0u && nb != 0x7f800000u;
    const auto put = [&](int i, const u32x4v (&v)[4]) {
        int g, c;
        place(i, g, c);
        unsigned code[2][4];                   // [four columns][row]
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const unsigned a = v[r][2 * q], b = v[r][2 * q + 1];
                if (fast) code[q][r] = Bits<T>::codes(a, b, now);
                else code[q][r] = codes2(Bits<T>::f(a & 0xffffu) / now, Bits<T>::f(a >> 16) / now) |
                                  codes2(Bits<T>::f(b & 0xffffu) / now, Bits<T>::f(b >> 16) / now) << 16;
            }
        const int first = 4 * g - off;         // run index of the group's first position
        if (KEYS) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (first + r >= 0 && first + r < n) *(u32x2*)(tile + (4 * g + r) * W + 8 * c) = u32x2{code[0][r], code[1][r]};
        } else {
            transpose4(code[0]);
            transpose4(code[1]);
            const bool whole = first >= 0 && first + 4 <= n;
#pragma unroll
            for (int col = 0; col < 8; ++col) {
                const unsigned w = code[col >> 2][col & 3];
                uint8_t* to = tile + (8 * c + col) * P + 4 * g;
                if (whole) *(unsigned*)to = w;
                else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (first + r >= 0 && first + r < n) to[r] = (uint8_t)(w >> (8 * r));
                }
            }
        }
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (tid + h * NT < items) put(tid + h * NT, held[h]);
    for (int i = tid + HOLD * NT; i < items; i += NT) {
        u32x4v v[4];
        load(i, v);
        put(i, v);
    }
}

template <typename T, int W, int HOLD>
__global__ __launch_bounds__(256) void cache_append_kernel(AppendParams p) {
    __shared__ unsigned shared_max[4];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // all windows of the keys, then of the values; the heads of a window side by side, which read neighbouring pieces of its rows (41.0 -> 39.7 us)
    const int half = (int)gridDim.x >> 1;
    const bool keys = (int)blockIdx.x < half;
    const int id = keys ? (int)blockIdx.x : (int)blockIdx.x - half, head = id % p.H;
    const int P = 1 << p.shift, t_first = id / p.H * p.window;
    // Every wave finds the window's runs by itself, from loads that are in flight together: for the window's tokens and the 128 behind them, whether a
    // token goes on from its predecessor; a token with a place that does not begins a run, and the ones behind its bit are its length (P <= 128).
    bool place[3], on[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int t = t_first + 64 * i + lane;
        const int slot = t < p.T ? p.slots[t] : -1, prev = t > 0 && t < p.T ? p.slots[t - 1] : -2;
        place[i] = slot >= 0 && slot < p.limit;
        on[i] = place[i] && prev >= 0 && prev + 1 == slot && (slot & (P - 1)) != 0;
    }
    unsigned long long begins = __ballot(place[0] && !on[0] && lane < p.window);
    const unsigned long long on0 = __ballot(on[0]), on1 = __ballot(on[1]), on2 = __ballot(on[2]);
    const bool few = __popcll(begins) <= 2;
    for (int r = 0; begins; ++r) {
        const int i = __builtin_ctzll(begins);
        begins &= begins - 1;
        const auto ones = [](unsigned long long m) { return ~m ? (int)__builtin_ctzll(~m) : 64; };
        int n = 1 + (i < 63 ? min(ones(on0 >> (i + 1)), 63 - i) : 0);
        if (n == 64 - i) {
            const int more = ones(on1);
            n += more;
            if (more == 64) n += ones(on2);
        }
        const bool together = few && n >= 16;     // (of several runs, or for a short one, a wave each: 512 tokens of one request 6.1 us, 10.5 without)
        if (!together && (r & 3) != wave) continue;
        const int t0 = t_first + i, slot = __builtin_amdgcn_readfirstlane(p.slots[t0]);
        const int64_t block = slot >> p.shift;
        const int off = slot & (P - 1);
        if (together) {
            if (keys) append_run<T, W, HOLD, true, 256>(p, t0, n, block, off, head, shared_max);
            else append_run<T, W, HOLD, false, 256>(p, t0, n, block, off, head, shared_max);
        } else {
            if (keys) append_run<T, W, HOLD, true, 64>(p, t0, n, block, off, head, shared_max);
            else append_run<T, W, HOLD, false, 64>(p, t0, n, block, off, head, shared_max);
        }
    }
}

}  // namespace

hipError_t launch_cache_tables(const TablesParams& p, hipStream_t stream) {
    hipError_t e = launch1((const void*)cache_tables_kernel, dim3(1), dim3(kScanThreads), 0, stream, p);
    if (e == hipSuccess && !p.fused && p.T > 0)
        e = launch1((const void*)cache_slots_kernel, dim3((unsigned)(p.T + kSlotThreads - 1) / kSlotThreads), dim3(kSlotThreads), 0, stream, p);
    return e;
}

hipError_t launch_cache_append(const AppendParams& p, int dtype, hipStream_t stream) {
    const dim3 grid((unsigned)((p.T + p.window - 1) / p.window) * 2u * (unsigned)p.H);
    const auto kernel = [&](auto t) {
        using T = decltype(t);
        const bool two = (p.W << p.shift) > 8192;
        return p.W == 64 ? (const void*)cache_append_kernel<T, 64, 1>
             : p.W == 128 ? (two ? (const void*)cache_append_kernel<T, 128, 2> : (const void*)cache_append_kernel<T, 128, 1>)
             : p.W == 192 ? (two ? (const void*)cache_append_kernel<T, 192, 2> : (const void*)cache_append_kernel<T, 192, 1>)
                          : (two ? (const void*)cache_append_kernel<T, 256, 2> : (const void*)cache_append_kernel<T, 256, 1>);
    };
    return launch1(dtype == 0 ? kernel(_Float16{}) : kernel(__bf16{}), grid, dim3(256), 0, stream, p);
}

}  // namespace fa
