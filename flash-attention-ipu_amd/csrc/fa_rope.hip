// Norm of every query and key head with the position rotation, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w,  out = turn(y):  a' = a cos - b sin,  b' = a sin + b cos  for the pairs (a, b) of the first R
//   columns - (i, i + R/2), or (2i, 2i + 1) when interleaved - and the columns behind them pass through.
//   backward: g = turn back(d out);  dw = sum over rows g x r;  t = g w;  dx = r (t - x r mean(t x r)).
//
// Bound: memory.  Forward reads and writes every value once; backward reads x and d out once and writes dx.  A row is held in the
// registers of a few lanes (8 for 128 columns of 16 bits), a run of 16 bytes of each half of the pairs per lane, so that both members of a
// pair are in one lane and the mean costs a lane exchange per halving.  A lane group takes HC heads of one token: cosines, sines and
// the position are fetched once for them and HC rows' loads are in flight together.  Sums, statistics and angles are 32-bit.
// dw has no atomics: a workgroup keeps its sum in registers over a fixed set of rows, writes one [D] row, and a second kernel adds the rows in order.
// Measured: [4, 32 + 8 heads, 4096, 128] bf16 61 us forward, 93 us backward, 5.4 TB/s each (a copy: 5.15; the weights' sums 5 us more); [3, 16 + 4, 4001, 64] f32
// 21.5 us; [64 tokens, 32 + 8, 128] 4.1 us.
// A position below 0 marks a row of padding: its outputs and gradients are zeros.  A position behind the table gives NaN.
#include <hip/hip_runtime.h>

#include "fa_cache.h"
#include "fa_params.h"

namespace fa {
namespace {

// runs of E columns that a lane holds: 16 bytes, so that every access of a wave is whole lines
template <typename T> constexpr int kRun = 16 / (int)sizeof(T);
template <typename T, int E> struct Vec { typedef T type __attribute__((ext_vector_type(E))); };

template <bool STREAM, typename T, int E>
__device__ __forceinline__ void load_run(const T* p, float (&f)[E]) {
    using V = typename Vec<T, E>::type;
    V v;
    if constexpr (STREAM) v = __builtin_nontemporal_load((const V*)p);
    else v = *(const V*)p;
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = (float)v[i];
}
template <bool STREAM, typename T, int E>
__device__ __forceinline__ void store_run(T* p, const float (&f)[E]) {
    using V = typename Vec<T, E>::type;
    V v;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (T)f[i];
    if constexpr (STREAM) __builtin_nontemporal_store(v, (V*)p);
    else *(V*)p = v;
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    const int v = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
    return x + __builtin_bit_cast(float, v);
}
// sum over aligned groups of N lanes, in every lane of the group; N <= 16 through DPP: neighbours, pairs, then mirrored halves (whose
// lanes hold equal sums by then, so that the mirror is as good as an exchange)
template <int N>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (N >= 2) x = dpp_add<0xB1>(x);     // quad_perm 1,0,3,2
    if constexpr (N >= 4) x = dpp_add<0x4E>(x);     // quad_perm 2,3,0,1
    if constexpr (N >= 8) x = dpp_add<0x141>(x);    // row_half_mirror
    if constexpr (N >= 16) x = dpp_add<0x140>(x);   // row_mirror
    if constexpr (N >= 32) x += __shfl_xor(x, 16);
    if constexpr (N >= 64) x += __shfl_xor(x, 32);
    return x;
}

// position of token (b, l): the table row, -1 for padding, table_rows for a position that the table lacks
__device__ __forceinline__ int64_t row_of(const RopeParams& p, int b, int l) {
    if (p.positions == nullptr) return l < p.table_rows ? l : p.table_rows;
    const int64_t at = (int64_t)b * p.pos_sb + l;
    const int64_t pos = p.pos64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
    return pos < 0 ? -1 : pos < p.table_rows ? pos : p.table_rows;
}

// the weights of columns c .. c + E - 1 (16-byte aligned; ones without weights)
template <typename T, int E>
__device__ __forceinline__ void weight_run(const RopeParams& p, const void* w, int c, float (&f)[E]) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = 1.0f;
    } else if (p.w_f32) load_run<false>((const float*)w + c, f);
    else load_run<false>((const T*)w + c, f);
}
template <typename T>
__device__ __forceinline__ float weight_at(const RopeParams& p, const void* w, int i) {
    return w == nullptr ? 1.0f : p.w_f32 ? ((const float*)w)[i] : (float)((const T*)w)[i];
}

// item -> (batch entry, row, first head); the heads of an item are `chunks` apart, so that neighbouring lane groups read neighbouring heads
__device__ __forceinline__ void item_of(const RopeSide& s, int L, unsigned item, int& b, int& l, int& c) {
    if (s.head_inner) {
        const unsigned tok = item / (unsigned)s.chunks;
        c = (int)(item - tok * (unsigned)s.chunks);
        b = (int)(tok / (unsigned)L);
        l = (int)(tok - (unsigned)b * (unsigned)L);
    } else {
        const unsigned bc = item / (unsigned)L;
        l = (int)(item - bc * (unsigned)L);
        b = (int)(bc / (unsigned)s.chunks);
        c = (int)(bc - (unsigned)b * (unsigned)s.chunks);
    }
}

// turn (sign = 1) or turn back (sign = -1) the pairs that a lane holds: f0, f1 are its two runs of columns
template <bool INTER, int E>
__device__ __forceinline__ void turn(float (&f0)[E], float (&f1)[E], const float (&c)[E], const float (&s)[E], float sign) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float& a = INTER ? (i < E / 2 ? f0[2 * i] : f1[2 * i - E]) : f0[i];
        float& b = INTER ? (i < E / 2 ? f0[2 * i + 1] : f1[2 * i + 1 - E]) : f1[i];
        const float sn = s[i] * sign, a0 = a, b0 = b;
        a = a0 * c[i] - b0 * sn;
        b = a0 * sn + b0 * c[i];
    }
}

// D = 2 E LPR, 16-byte rows, R a multiple of 16.  STREAM: the launch moves more than the last cache holds, so that nothing is kept in it (rope_shape)
template <typename T, int LPR, bool INTER, int HC, bool BWD, bool STREAM>
__global__ __launch_bounds__(256) void rope_vec_kernel(RopeParams p) {
    const int which = (int)blockIdx.x >= p.side[0].blocks;
    const RopeSide& s = p.side[which];
    const int block = which ? (int)blockIdx.x - p.side[0].blocks : (int)blockIdx.x;
    constexpr int E = kRun<T>, D = 2 * E * LPR, GROUPS = 256 / LPR;
    const int j = (int)threadIdx.x % LPR, group = (int)threadIdx.x / LPR;
    const int R = p.R, rot = R / (2 * E);
    const bool rotated = j < rot;
    int c0, c1;             // the lane's two runs of columns
    if (INTER) {
        c0 = 2 * E * j;
        c1 = c0 + E;
    } else if (rotated) {
        c0 = E * j;
        c1 = R / 2 + E * j;
    } else {
        c0 = R + E * (j - rot);
        c1 = R + (D - R) / 2 + E * (j - rot);
    }
    float w0[E], w1[E], dw0[E], dw1[E];
    weight_run<T>(p, s.w, c0, w0);
    weight_run<T>(p, s.w, c1, w1);
#pragma unroll
    for (int i = 0; i < E; ++i) dw0[i] = dw1[i] = 0.f;
    const T* x = (const T*)s.x;
    const T* dy = (const T*)s.dy;
    T* y = (T*)s.y;
    for (int item = block * GROUPS + group; item < s.items; item += s.blocks * GROUPS) {
        int b, l, c;
        item_of(s, p.L, (unsigned)item, b, l, c);
        const int64_t pos = row_of(p, b, l);
        float f0[HC][E], f1[HC][E], g0[HC][E], g1[HC][E], cs[E], sn[E];
#pragma unroll
        for (int h = 0; h < HC; ++h) {
            const int head = c + h * s.chunks;
            if (head < s.heads) {
                const T* row = x + (int64_t)b * s.x_sb + (int64_t)head * s.x_sh + (int64_t)l * s.x_sl;
                load_run<STREAM>(row + c0, f0[h]);
                load_run<STREAM>(row + c1, f1[h]);
                if constexpr (BWD) {
                    const T* drow = dy + (int64_t)b * s.dy_sb + (int64_t)head * s.dy_sh + (int64_t)l * s.dy_sl;
                    load_run<STREAM>(drow + c0, g0[h]);
                    load_run<STREAM>(drow + c1, g1[h]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
        const bool pad = pos < 0;
        if (rotated && pos >= 0 && pos < p.table_rows) {
            const float* t = p.table + pos * R + E * j;
            load_run<false>(t, cs);
            load_run<false>(t + R / 2, sn);
        }
        if (pos == p.table_rows) {
#pragma unroll
            for (int i = 0; i < E; ++i) cs[i] = sn[i] = __builtin_nanf("");
        }
#pragma unroll
        for (int h = 0; h < HC; ++h) {
            const int head = c + h * s.chunks;
            if (head >= s.heads) continue;
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) sq += f0[h][i] * f0[h][i];
#pragma unroll
            for (int i = 0; i < E; ++i) sq += f1[h][i] * f1[h][i];
            const float r = rsqrtf(group_sum<LPR>(sq) * (1.0f / D) + p.eps);
            float o0[E], o1[E];
            if constexpr (!BWD) {
#pragma unroll
                for (int i = 0; i < E; ++i) { o0[i] = f0[h][i] * r * w0[i]; o1[i] = f1[h][i] * r * w1[i]; }
                turn<INTER>(o0, o1, cs, sn, 1.f);
            } else {
                turn<INTER>(g0[h], g1[h], cs, sn, -1.f);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float h0 = f0[h][i] * r, h1 = f1[h][i] * r;
                    if (!pad) { dw0[i] += g0[h][i] * h0; dw1[i] += g1[h][i] * h1; }
                    o0[i] = g0[h][i] * w0[i];
                    o1[i] = g1[h][i] * w1[i];
                    dot += o0[i] * h0 + o1[i] * h1;
                    f0[h][i] = h0;
                    f1[h][i] = h1;
                }
                const float m = group_sum<LPR>(dot) * (1.0f / D);
#pragma unroll
                for (int i = 0; i < E; ++i) { o0[i] = r * (o0[i] - f0[h][i] * m); o1[i] = r * (o1[i] - f1[h][i] * m); }
            }
            if (pad) {
#pragma unroll
                for (int i = 0; i < E; ++i) o0[i] = o1[i] = 0.f;
            }
            T* row = y + (int64_t)b * s.y_sb + (int64_t)head * s.y_sh + (int64_t)l * s.y_sl;
            store_run<STREAM>(row + c0, o0);
            store_run<STREAM>(row + c1, o1);
        }
    }
    if constexpr (BWD) {
        if (s.dw_part == nullptr) return;
        // the wave's lane groups, then the four waves, in a fixed order
        __shared__ float part[4][D];
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < E; ++i) {
#pragma unroll
            for (int d = LPR; d < 64; d *= 2) {
                dw0[i] += __shfl_xor(dw0[i], d);
                dw1[i] += __shfl_xor(dw1[i], d);
            }
        }
        if (lane < LPR) {
#pragma unroll
            for (int i = 0; i < E; ++i) { part[wave][c0 + i] = dw0[i]; part[wave][c1 + i] = dw1[i]; }
        }
        __syncthreads();
        for (int d = (int)threadIdx.x; d < D; d += 256) s.dw_part[(int64_t)block * D + d] = part[0][d] + part[1][d] + part[2][d] + part[3][d];
    }
}

// any even D <= 512, any strides and alignment: one wave per row, a pair per lane and step
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeParams p) {
    const int which = (int)blockIdx.x >= p.side[0].blocks;
    const RopeSide& s = p.side[which];
    const int block = which ? (int)blockIdx.x - p.side[0].blocks : (int)blockIdx.x;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int D = p.D, R = p.R, half = R / 2;
    constexpr int N = 4;    // pairs per lane
    int ca[N], cb[N];
    float wa[N], wb[N], dwa[N], dwb[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = lane + 64 * n;
        if (p.interleaved) { ca[n] = 2 * i; cb[n] = 2 * i + 1; }
        else if (i < half) { ca[n] = i; cb[n] = i + half; }
        else { ca[n] = R + (i - half); cb[n] = R + (D - R) / 2 + (i - half); }
        const bool in = 2 * i < D;
        wa[n] = in ? weight_at<T>(p, s.w, ca[n]) : 0.f;
        wb[n] = in ? weight_at<T>(p, s.w, cb[n]) : 0.f;
        dwa[n] = dwb[n] = 0.f;
    }
    for (int item = block * 4 + wave; item < s.items; item += s.blocks * 4) {
        int b, l, c;
        item_of(s, p.L, (unsigned)item, b, l, c);      // (heads per group is 1 here: c is the head)
        const int64_t pos = row_of(p, b, l);
        const T* row = (const T*)s.x + (int64_t)b * s.x_sb + (int64_t)c * s.x_sh + (int64_t)l * s.x_sl;
        const T* drow = BWD ? (const T*)s.dy + (int64_t)b * s.dy_sb + (int64_t)c * s.dy_sh + (int64_t)l * s.dy_sl : nullptr;
        T* out = (T*)s.y + (int64_t)b * s.y_sb + (int64_t)c * s.y_sh + (int64_t)l * s.y_sl;
        float a[N], bb[N], sq = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool in = 2 * (lane + 64 * n) < D;
            a[n] = in ? (float)row[ca[n]] : 0.f;
            bb[n] = in ? (float)row[cb[n]] : 0.f;
            sq += a[n] * a[n] + bb[n] * bb[n];
        }
        const float r = rsqrtf(group_sum<64>(sq) / (float)D + p.eps);
        float oa[N], ob[N], dot = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = lane + 64 * n;
            float cs = 1.f, sn = 0.f;
            if (i < half && pos >= 0 && pos < p.table_rows) { cs = p.table[pos * R + i]; sn = p.table[pos * R + half + i]; }
            if (pos == p.table_rows) cs = sn = __builtin_nanf("");
            if constexpr (!BWD) {
                const float u = a[n] * r * wa[n], v = bb[n] * r * wb[n];
                oa[n] = u * cs - v * sn;
                ob[n] = u * sn + v * cs;
            } else {
                const bool in = 2 * i < D;
                const float du = in ? (float)drow[ca[n]] : 0.f, dv = in ? (float)drow[cb[n]] : 0.f;
                const float ga = du * cs + dv * sn, gb = dv * cs - du * sn;
                a[n] *= r;
                bb[n] *= r;
                if (pos >= 0) { dwa[n] += ga * a[n]; dwb[n] += gb * bb[n]; }
                oa[n] = ga * wa[n];
                ob[n] = gb * wb[n];
                dot += in ? oa[n] * a[n] + ob[n] * bb[n] : 0.f;
            }
        }
        if constexpr (BWD) {
            const float m = group_sum<64>(dot) / (float)D;
#pragma unroll
            for (int n = 0; n < N; ++n) { oa[n] = r * (oa[n] - a[n] * m); ob[n] = r * (ob[n] - bb[n] * m); }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (2 * (lane + 64 * n) >= D) continue;
            out[ca[n]] = (T)(pos < 0 ? 0.f : oa[n]);
            out[cb[n]] = (T)(pos < 0 ? 0.f : ob[n]);
        }
    }
    if constexpr (BWD) {
        if (s.dw_part == nullptr) return;
        __shared__ float part[4][512];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (2 * (lane + 64 * n) >= D) continue;
            part[wave][ca[n]] = dwa[n];
            part[wave][cb[n]] = dwb[n];
        }
        __syncthreads();
        for (int d = (int)threadIdx.x; d < D; d += 256) s.dw_part[(int64_t)block * D + d] = part[0][d] + part[1][d] + part[2][d] + part[3][d];
    }
}

// dw = sum of the workgroups' rows in a fixed order: 64 columns per workgroup, 32 strands of rows, whose loads are independent and in flight together (the
// kernel is a few microseconds of latency)
constexpr int kDwStrands = 32;
template <typename T>
__global__ __launch_bounds__(1024) void rope_dw_kernel(RopeParams p) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const RopeSide& s = p.side[blockIdx.y];
    if (s.dw == nullptr) return;
    const int tid = (int)threadIdx.x, c = tid & 31, strand = tid >> 5, col = (int)blockIdx.x * 64 + 2 * c;
    __shared__ f32x2 part[16][32];
    f32x2 sum = {0.f, 0.f};
    if (col < p.D) {
#pragma unroll 8
        for (int r = strand; r < s.blocks; r += kDwStrands) sum += *(const f32x2*)(s.dw_part + (int64_t)r * p.D + col);
    }
    sum[0] += __shfl_xor(sum[0], 32);
    sum[1] += __shfl_xor(sum[1], 32);
    if ((strand & 1) == 0) part[strand >> 1][c] = sum;
    __syncthreads();
    if (tid < 32 && col < p.D) {
        sum = part[0][c];
#pragma unroll
        for (int r = 1; r < 16; ++r) sum += part[r][c];
        if (p.w_f32) {
            ((float*)s.dw)[col] = sum[0];
            ((float*)s.dw)[col + 1] = sum[1];
        } else {
            ((T*)s.dw)[col] = (T)sum[0];
            ((T*)s.dw)[col + 1] = (T)sum[1];
        }
    }
}

template <typename T, int LPR, bool INTER, bool BWD>
const void* vec_kernel(int hc, bool stream) {
    return hc == 1 ? (const void*)rope_vec_kernel<T, LPR, INTER, 1, BWD, false>
         : stream ? (const void*)rope_vec_kernel<T, LPR, INTER, 2, BWD, true> : (const void*)rope_vec_kernel<T, LPR, INTER, 2, BWD, false>;
}
template <typename T, bool INTER, bool BWD>
const void* vec_kernel(int D, int hc, bool stream) {
    constexpr int L = 16 / kRun<T>;          // lanes of 32 columns
    return D == 32 ? vec_kernel<T, L, INTER, BWD>(hc, stream) : D == 64 ? vec_kernel<T, 2 * L, INTER, BWD>(hc, stream)
         : D == 128 ? vec_kernel<T, 4 * L, INTER, BWD>(hc, stream) : vec_kernel<T, 8 * L, INTER, BWD>(hc, stream);
}
template <typename T, bool BWD>
hipError_t launch_rope(const RopeParams& p, bool vec, int hc, bool nt, hipStream_t stream) {
    const dim3 grid((unsigned)(p.side[0].blocks + p.side[1].blocks));
    const void* k = !vec ? (const void*)rope_any_kernel<T, BWD> : p.interleaved ? vec_kernel<T, true, BWD>(p.D, hc, nt) : vec_kernel<T, false, BWD>(p.D, hc, nt);
    hipError_t e = launch1(k, grid, dim3(256), 0, stream, p);
    if (e == hipSuccess && BWD && (p.side[0].dw || p.side[1].dw))
        e = launch1((const void*)rope_dw_kernel<T>, dim3((unsigned)(p.D + 63) / 64, 2), dim3(1024), 0, stream, p);
    return e;
}

}  // namespace

hipError_t launch_rope_fwd(const RopeParams& p, int dtype, bool vec, int hc, bool nt, hipStream_t stream) {
    return dtype == 0 ? launch_rope<_Float16, false>(p, vec, hc, nt, stream) : dtype == 1 ? launch_rope<__bf16, false>(p, vec, hc, nt, stream)
                                                                                      : launch_rope<float, false>(p, vec, hc, nt, stream);
}
hipError_t launch_rope_bwd(const RopeParams& p, int dtype, bool vec, int hc, bool nt, hipStream_t stream) {
    return dtype == 0 ? launch_rope<_Float16, true>(p, vec, hc, nt, stream) : dtype == 1 ? launch_rope<__bf16, true>(p, vec, hc, nt, stream)
                                                                                     : launch_rope<float, true>(p, vec, hc, nt, stream);
}

}  // namespace fa
