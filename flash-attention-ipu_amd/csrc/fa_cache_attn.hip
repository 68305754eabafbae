// Causal attention of ragged query runs over a block cache of e4m3 codes with one scale per block and head (fa_cache.h: layout).
//
//   request b: n = cu_q[b+1] - cu_q[b] query tokens, the last n of its len = seq_lens[b] tokens; token i sees the keys below limit = len - n + i + 1.
//   S = scale (q . code_k) scale_k,  O = sum_k exp(S - max) scale_v code_v / sum_k exp(S - max);  a row that sees no key gives zeros.
//
// Query rows of one key/value head are packed (token, head of its group), token first, so that a grouped head's codes are read and
// converted once for all its query heads.  The unit of work is 64 tokens.  Products run transposed on v_mfma_f32_16x16x32, S^T = K Q^T and
// O^T = V^T P^T: a query row is a lane's column, so that its maximum, sum and rescale are per-lane values, and the layouts are chosen so that nothing
// moves between lanes on the way:
//   * row `r` of key tile t (16 keys) is key 16 (r >> 2) + 4 t + (r & 3) of the unit: a lane's four results of the four tiles are the sixteen
//     CONSECUTIVE keys 16 (lane >> 4) .. + 15, which is what the B operand of the second product wants of that lane (two products of 32 keys);
//   * the value cache is token-inner, so the matching A operand (column d, those sixteen keys) is one 16-byte load, as is a key row's share.
// e4m3 -> 16-bit is exact, one instruction per two values.  Scales cost no instruction per score: scale_k and the softmax scale are the factor
// of the exponent's fma, and the weight that meets the codes of V is P' = P scale_v = 2^(s kf + log2(scale_v) - max), rounded once to the operand type; the
// sum of the weights takes a lane's sum of P' (bf16: rounded) over scale_v, once per unit.  `max` is the row's largest score for bf16, whose exponents reach as
// far as 32-bit ones.  f16 weights have thirty binades and ten of subnormals, and a row's scales may differ by more: its `max` is the largest s kf + log2(scale_v)
// of the keys that the row sees, less kLift, so that the largest P' stays near the type's top and what vanishes is 2^-32 of the row's own largest term,
// whatever the scales of blocks are that it does not see or gives no weight.  Maximum, sum and O are 32-bit.
//
// Two kernels:
//   row kernel   few rows per key/value head (a decoding step): bound by the cache's bytes.  Codes go from memory straight into
//                registers; a wave takes every fourth unit, the next unit's loads are in flight under the current one's arithmetic.  The
//                grid is fixed; the units of all (request, head, row tile) are one line that is cut into equal ranges on the device, from the
//                lengths there: no length is known to the host, and one long request fills the chip.  A (request, head, row tile) inside one range
//                is finished there; one that crosses ranges leaves unnormalised partial sums that the join kernel adds in order.
//                64 requests of 4600 tokens on average, 8 heads of 128: 105 us = 5.7 TB/s, every code read once, and 5 us for the join.
//   tile kernel  128 rows per workgroup, 64 where no request has more (prompts): bound by the matrix pipe.  Four waves share a unit's operands,
//                converted once into LDS in the very order in which the lanes read them.  Grids too small for the chip cut every tile's
//                key range into `splits` parts.  Four prompts of 2048 over 8192 tokens, 32 / 8 heads: bf16 1020 TFLOP/s at width 128, 700 at 64, 600 at 192, 640 at 256 (f16 1000, 685, 560, 590)
//                (matrix pipe 39 % busy, vector issue 41 %, LDS 51 %).
// Stale codes behind a request's end are cleared before they meet a zero weight (0 * NaN), and a NaN code that only some rows of a unit may
// see reaches those rows alone.
#include <hip/hip_runtime.h>

#include "fa_cache.h"
#include "fa_device.h"

namespace fa {
namespace {

typedef unsigned u32x2c __attribute__((ext_vector_type(2)));
typedef float f32x2c __attribute__((ext_vector_type(2)));

template <typename T> struct Code;
template <> struct Code<__bf16> {
    static __device__ __forceinline__ unsigned lo(unsigned w) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)); }
    static __device__ __forceinline__ unsigned hi(unsigned w) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)); }
};
template <> struct Code<_Float16> {
    static __device__ __forceinline__ unsigned lo(unsigned w) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)); }
    static __device__ __forceinline__ unsigned hi(unsigned w) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)); }
};
// eight codes -> one operand fragment
template <typename T>
__device__ __forceinline__ typename Elt<T>::vec8 fragment(unsigned a, unsigned b) {
    const u32x4 v = {Code<T>::lo(a), Code<T>::hi(a), Code<T>::lo(b), Code<T>::hi(b)};
    return __builtin_bit_cast(typename Elt<T>::vec8, v);
}
template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    typedef T vec2 __attribute__((ext_vector_type(2)));
    const vec2 v = {(T)a, (T)b};
    return __builtin_bit_cast(unsigned, v);
}
// the four 16-lane groups of a wave hold parts of the same 16 rows: maximum / sum over the groups, in every lane
__device__ __forceinline__ HalfPair group_exchange(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return {__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)};
}
__device__ __forceinline__ float rows_max(float x) {
    const HalfPair p = group_exchange(x);
    x = __builtin_fmaxf(p.lo, p.hi);
    const HalfPair h = half_exchange(x);
    return __builtin_fmaxf(h.lo, h.hi);
}
__device__ __forceinline__ float rows_sum(float x) {
    const HalfPair p = group_exchange(x);
    x = p.lo + p.hi;
    const HalfPair h = half_exchange(x);
    return h.lo + h.hi;
}
// codes of the keys at and behind `valid` (of the sixteen in v) cleared
__device__ __forceinline__ u32x4 clear_behind(u32x4 v, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = valid - 4 * i;
        v[i] = n >= 4 ? v[i] : n <= 0 ? 0u : v[i] & (0xffffffffu >> (8 * (4 - n)));
    }
    return v;
}

__device__ __forceinline__ bool has_nan(u32x4 v) {
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= ((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return any != 0;
}
// the NaN codes of v cleared; which of the sixteen they were
__device__ __forceinline__ unsigned take_nan(u32x4& v) {
    unsigned bits = 0;
    asm volatile("" : "+v"(v));                // (else has_nan's terms are kept for all of a lane's codes)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned n = (((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;     // 1 in every NaN byte
        v[i] &= ~(n * 0xffu);
        bits |= ((n | n >> 7 | n >> 14 | n >> 21) & 0xfu) << (4 * i);
    }
    return bits;
}

// Tables, lengths and scales do not change while a kernel runs: read through the constant address space, uniform ones stay scalar loads behind a barrier (the
// compiler takes a barrier for a change of all memory, and would wait for the codes in flight with every vector load in their place).
template <typename V>
__device__ __forceinline__ V constant(const V* p) {
    return *(const __attribute__((address_space(4))) V*)(unsigned long long)p;
}

// ---- a request as every kernel here sees it: all indexes held inside what the caller's tensors have ----------------------------------------
struct Request {
    int first, n, len, units;
};
__device__ __forceinline__ Request request_of(const CacheAttnParams& p, int b) {
    Request r;
    const int a = min(max(constant(p.cu_q + b), 0), p.T), e = min(max(constant(p.cu_q + b + 1), a), p.T);
    const long long room = (long long)p.width << p.shift;
    r.first = a;
    r.n = e - a;
    r.len = max(constant(p.seq_lens + b), 0);
    r.len = r.len < room ? r.len : (int)room;
    if (p.granted && constant(p.granted + b) <= 0) r.len = 0;      // (rows whose own tokens are not in the cache)
    r.units = max(1, (int)(((long long)r.len + 63) >> 6));
    return r;
}

__device__ __forceinline__ long long uniform(long long x) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)x), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ long long lane_value(long long x, int lane) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)x, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(x >> 32), lane);
    return (long long)((unsigned long long)hi << 32 | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ long long sum_step(long long x) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false), hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
    return x + (long long)((unsigned long long)hi << 32 | lo);
}
// Every wave finds its place by itself, without a barrier: `items` summed over the requests (each lane a stretch of them), `want(total)` names the item to
// find, and the stretch that holds it is walked.  prefix (or null) receives the sums.  The request comes with it: a small call is a chain of loads.
struct Place {
    Request rq;
    int b;
    long long off, total;
};
template <typename Items, typename Want>
__device__ __forceinline__ Place find_place(const CacheAttnParams& p, Items items, Want want, long long* prefix) {
    const int lane = (int)threadIdx.x & 63, per = (p.B + 63) >> 6, from = min(lane * per, p.B), to = min(from + per, p.B);
    Place f{};
    long long mine = 0;
    for (int b = from; b < to; ++b) {
        f.rq = request_of(p, b);
        mine += items(f.rq);
    }
    long long incl = mine;
    incl = sum_step<0x111, 0xf>(incl);      // row_shr 1, 2, 4, 8; then the rows' last lanes onto the rows behind them
    incl = sum_step<0x112, 0xf>(incl);
    incl = sum_step<0x114, 0xf>(incl);
    incl = sum_step<0x118, 0xf>(incl);
    incl = sum_step<0x142, 0xa>(incl);
    incl = sum_step<0x143, 0xc>(incl);
    const long long before = incl - mine;
    f.total = lane_value(incl, 63);
    const long long x = want(f.total);
    const bool here = x >= before && x < incl;
    f.b = from;
    f.off = x - before;
    if (here && per > 1)
        for (;; ++f.b) {
            f.rq = request_of(p, f.b);
            const long long n = items(f.rq);
            if (f.off < n) break;
            f.off -= n;
        }
    if (prefix) {
        long long at = before;
        for (int b = from; b < to; ++b) { prefix[b] = at; at += items(request_of(p, b)); }
        if (lane == 0) prefix[p.B] = f.total;
    }
    const unsigned long long who = __ballot(here);
    const int lead = who ? (int)__builtin_ctzll(who) : 0;      // (no lane: the item lies behind the last one, and the caller goes home)
    f.b = __builtin_amdgcn_readlane(f.b, lead);
    f.off = lane_value(f.off, lead);
    f.rq.first = __builtin_amdgcn_readlane(f.rq.first, lead);
    f.rq.n = __builtin_amdgcn_readlane(f.rq.n, lead);
    f.rq.len = __builtin_amdgcn_readlane(f.rq.len, lead);
    f.rq.units = __builtin_amdgcn_readlane(f.rq.units, lead);
    return f;
}

// a value that the compiler may not form ahead of its use: what is derived from it is not kept in registers round a loop
__device__ __forceinline__ int fresh_scalar(int x) { asm volatile("" : "+s"(x)); return x; }
__device__ __forceinline__ int fresh_lane(int x) { asm volatile("" : "+v"(x)); return x; }

// LDS traffic between the lanes of one wave: what stands before is done before what stands behind (the hardware keeps a wave's order; the compiler has to)
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- the arithmetic of one unit for the 16 NR rows of a wave --------------------------------------------------------------------------------
template <typename T, int W, int NR>
struct RowState {
    static constexpr int NC = W / 32, ND = W / 16;       // k-steps of Q K^T; 16-column tiles of O
    using vec8 = typename Elt<T>::vec8;
    vec8 q[NR][NC];
    f32x4 o[NR][ND];
    float m[NR], l[NR];
    int limit[NR];                                       // keys that the lane's row sees
    int limit_min;                                       // over the wave's rows (uniform)
    using NanBits = typename std::conditional<W <= 128, unsigned, unsigned long long>::type;
    NanBits nan[NR];                                     // bit 4 d + i: o[r][d][i] saw a NaN value (note_nan)

    // f16: with weights up to 2^(kSlack + kLift) = 2^15 the largest stay inside the type
    static constexpr bool kHalf = Elt<T>::is_f16;
    static constexpr float kSlack = 8.f, kLift = kHalf ? 7.f : 0.f;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            nan[r] = 0;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // rows row0 .. row0 + 16 NR - 1 of (request, key/value head h)
    __device__ __forceinline__ void load(const CacheAttnParams& p, const Request& rq, int h, int row0, int lane) {
        const int col = lane & 15, lg = lane >> 4, rows = rq.n * p.group;
        limit_min = rq.len - rq.n + row0 / p.group + 1;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = row0 + 16 * r + col;
            const bool in = row < rows;
            const int i = in ? row / p.group : 0, g = in ? row - i * p.group : 0;
            limit[r] = in ? rq.len - rq.n + i + 1 : limit_min;
            const T* src = (const T*)p.q + (int64_t)(rq.first + i) * p.q_st + (int64_t)(h * p.group + g) * p.q_sh;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 64 * (c >> 1) + 16 * lg + 8 * (c & 1);
                u32x4 v = {0, 0, 0, 0};
                if (in && d < p.D) v = *(const u32x4*)(src + d);
                q[r][c] = __builtin_bit_cast(vec8, v);
            }
        }
    }
    // S^T of a unit.  key(t, c): fragment c of key tile t.  FENCE: key tiles one after the other - where `key` converts, the compiler would otherwise
    // convert all of them first and spill
    template <bool FENCE, typename Key>
    __device__ __forceinline__ void scores(Key key, f32x4 (&s)[NR][4]) const {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int r = 0; r < NR; ++r) s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const vec8 a = key(t, c);
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r][t] = Elt<T>::mfma16(a, q[r][c], s[r][t]);
            }
            if (FENCE) __builtin_amdgcn_sched_barrier(0);
        }
    }
    // scores that a row may not see; the lane's keys are key0 .. key0 + 15, dead: they have no block
    __device__ __forceinline__ void mask(f32x4 (&s)[NR][4], int key0, bool dead) const {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int see = dead ? 0 : limit[r] - key0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][t][i] = 4 * t + i < see ? s[r][t][i] : -INFINITY;
        }
    }
    // The value scale that the weights carry.  f16: one below 2^-64 counts as 2^-64 (448 times that is far below half of the smallest f16 output), so that P' of a block
    // of zeros beside large values does not leave 32-bit floats, and its weights stay in the sum.
    static __device__ __forceinline__ float carried(float vs) { return kHalf ? __builtin_fmaxf(vs, 0x1p-64f) : vs; }
    // every row's largest exponent of the unit: score, f16 with the value scale.  kf: scale_k times the softmax scale; vs: the lane's value scale
    __device__ __forceinline__ void peak(const f32x4 (&s)[NR][4], float kf, float vs, float (&top)[NR]) const {
        const float lift = kHalf ? __builtin_amdgcn_logf(carried(vs)) : 0.f;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float x = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; i += 2) x = __builtin_fmaxf(__builtin_fmaxf(x, s[r][t][i]), s[r][t][i + 1]);
            top[r] = rows_max(kHalf ? __builtin_fmaf(x, kf, lift) : x * kf);
        }
    }
    // the reference maximum goes up where an exponent would leave 2^kSlack above it (weights up to 2^kSlack round as well as weights up to 1); most units do not
    // pay for the rescale
    __device__ __forceinline__ void raise(const float (&top)[NR]) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (__any(top[r] > m[r] + kSlack)) {
                const float now = __builtin_fmaxf(m[r], top[r]), alpha = fast_exp2(m[r] - (now == -INFINITY ? 0.f : now));
                l[r] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[r][d] *= alpha;
                m[r] = now;
            }
        }
    }
    // P' of a unit, and its sum into l.  vs: the lane's value scale
    __device__ __forceinline__ void weights(const f32x4 (&s)[NR][4], vec8 (&w)[NR][2], float kf, float vs) {
        vs = carried(vs);
        const float shift = __builtin_amdgcn_logf(vs) + kLift, back = __builtin_amdgcn_rcpf(vs);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float base = shift - (m[r] == -INFINITY ? 0.f : m[r]);
            float sum[2] = {0.f, 0.f};
            unsigned u[8];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = fast_exp2(__builtin_fmaf(s[r][t][i], kf, base));
                    if constexpr (kHalf) sum[i & 1] += e[i];
                }
                u[2 * t] = pack2<T>(e[0], e[1]);
                u[2 * t + 1] = pack2<T>(e[2], e[3]);
                // bf16: one instruction adds two rounded weights (width 256, prompts of 2048 over 8192: 4190 -> 3900 us, width 192 3275 -> 3105, width 128 1 % or less).
                // They are the weights that the values meet, so that the quotient is a mean with weights that add up to one: its error is no larger than with the sum of
                // the unrounded ones (512 normal scores, against 64 bits: mean 1.3e-4 of sum p |v| and 1.5e-4).  f16 weights of small value scales round to zero and
                // still count in the sum: they are added before they are rounded.
                if constexpr (!kHalf) {
                    typedef __bf16 vec2 __attribute__((ext_vector_type(2)));
                    const vec2 one = {(__bf16)1.0f, (__bf16)1.0f};
                    sum[0] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(vec2, u[2 * t]), one, sum[0], false);
                    sum[1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(vec2, u[2 * t + 1]), one, sum[1], false);
                }
            }
            l[r] = __builtin_fmaf(sum[0] + sum[1], back, l[r]);
            asm volatile("" : "+v"(l[r]));            // (here: moved behind the products, the sum would keep every weight in a register)
            const u32x4 a = {u[0], u[1], u[2], u[3]}, b = {u[4], u[5], u[6], u[7]};
            w[r][0] = __builtin_bit_cast(vec8, a);
            w[r][1] = __builtin_bit_cast(vec8, b);
        }
    }
    // O^T += V^T P'^T for the column tiles D0 .. D1 - 1.  value(d, u): fragment of columns 16 d .., keys 8 u .. + 7 of every lane's sixteen
    template <int D0, int D1, bool FENCE, typename Value>
    __device__ __forceinline__ void values(Value value, const vec8 (&w)[NR][2]) {
        if (FENCE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = D0; d < D1; ++d) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const vec8 a = value(d, u);
#pragma unroll
                for (int r = 0; r < NR; ++r) o[r][d] = Elt<T>::mfma16(a, w[r][u], o[r][d]);
            }
            if (FENCE && (NR * W > 128 || d % 2)) __builtin_amdgcn_sched_barrier(0);
        }
    }
    // A unit that some rows see only in part holds NaN values: they were taken out of the operands (take_nan) and are noted for the rows that see
    // them; keys[4 column ..]: the unit's keys with NaN in that column, sixteen in each of four.  Other lanes wrote them: the caller orders that (wave_order, or a barrier)
    __device__ __forceinline__ void note_nan(const unsigned short* keys, int unit, int lg) {
        keys += 16 * fresh_lane(lg);
#pragma unroll 1
        for (int e = 0; e < 4 * ND; ++e) {
            unsigned long long k;
            __builtin_memcpy(&k, __builtin_assume_aligned(keys + 4 * (16 * (e >> 2) + (e & 3)), 8), 8);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int see = limit[r] - 64 * unit;
                const unsigned long long seen = see <= 0 ? 0ull : see >= 64 ? ~0ull : (1ull << see) - 1;
                nan[r] |= (NanBits)((k & seen) != 0) << e;
            }
        }
    }
    // the segment's end: NaN where it was seen
    __device__ __forceinline__ void put_nan() {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (!__any(nan[r] != 0)) continue;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][d][i] = (nan[r] >> (4 * d + i)) & 1 ? __builtin_nanf("") : o[r][d][i];
        }
    }
    // O / l of rows row0 .. into the output
    __device__ __forceinline__ void store(const CacheAttnParams& p, const Request& rq, int h, int row0, int lane, const float (&sum)[NR]) const {
        const int col = lane & 15, lg = lane >> 4, rows = rq.n * p.group;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = row0 + 16 * r + col;
            if (row >= rows) continue;
            const int i = row / p.group, g = row - i * p.group;
            T* dst = (T*)p.o + (int64_t)(rq.first + i) * p.o_st + (int64_t)(h * p.group + g) * p.o_sh;
            const float inv = sum[r] == 0.f ? 0.f : 1.0f / sum[r];
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int at = 16 * d + 4 * lg;
                if (at >= p.D) continue;
                const f32x4 v = o[r][d] * inv;
                *(u32x2c*)(dst + at) = u32x2c{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            }
        }
    }
    // unnormalised sums into a workspace slot of `rows16` rows, from its row `at` on
    __device__ __forceinline__ void park(const CacheAttnParams& p, long long slot, int rows16, int at, int lane, const float (&sum)[NR], const float (&top)[NR]) const {
        const int col = lane & 15, lg = lane >> 4;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const long long row = slot * rows16 + at + 16 * r + col;
            if (lg == 0) { p.ws_ml[2 * row] = top[r]; p.ws_ml[2 * row + 1] = sum[r]; }
#pragma unroll
            for (int d = 0; d < ND; ++d) *(f32x4*)(p.ws_o + row * W + 16 * d + 4 * lg) = o[r][d];
        }
    }
};

// the block of a token index, -1 where the table has none that exists
__device__ __forceinline__ int block_at(const CacheAttnParams& p, const int* table, int index) {
    const int id = index < p.width ? constant(table + index) : -1;
    return (unsigned)id < (unsigned)p.num_blocks ? id : -1;
}

// Where a lane finds its codes of a unit, the scales, and whether its keys exist.  Blocks of a unit and more: base addresses are uniform and the
// lane's part is a 32-bit offset that all units share; smaller blocks: the lane's own addresses.
template <bool SMALL>
struct UnitAt {
    const uint8_t* k;
    const uint8_t* v;
    float kf, vs;             // the lane's factors: scale_k times the softmax scale, the value scale
    bool dead, none;          // the lane's sixteen keys have no block; the unit has none at all (uniform)
    bool blank;               // their values count as zeros: no block, or a scale of zero
    // (a scale of zero, or none, becomes one that makes everything vanish but leaves no 0 * inf)
    static __device__ __forceinline__ float factor(float x) { return __builtin_fmaxf(x, 0x1p-100f); }
    __device__ __forceinline__ void find(const CacheAttnParams& p, const int* table, int len, int u, int h, int W, int lane) {
        const int lg = lane >> 4, wk = lane & 15, P = 1 << p.shift, first = 64 * u;
        if constexpr (!SMALL) {
            const int id = first < len ? block_at(p, table, first >> p.shift) : -1;
            none = id < 0;
            dead = none;
            const long long blk = none ? 0 : id;
            const int in = first & (P - 1);
            k = p.k + blk * p.k_bs + (int64_t)(h * P + in) * W;
            v = p.v + blk * p.v_bs + (int64_t)h * P * W + in;
            kf = factor(none ? 0.f : constant(p.ks + blk * p.ks_bs + h) * p.scale_log2);
            vs = none ? 0.f : constant(p.vs + blk * p.vs_bs + h);
            blank = vs == 0.f;
            vs = factor(vs);
        } else {
            const int kk = first + 16 * (wk >> 2), vk = first + 16 * lg;
            // The blocks of the unit's sixteen-key pieces are uniform: scalar loads.  (As the lanes' own loads they would come behind the codes in flight, and every
            // unit would wait for them: 64 requests of 4096, blocks of 16: width 64 54 us, so 48; width 128 99 and 94.  The scales as scalar loads too: 63 and 102.)
            int ids[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = first + 16 * j, index = key >> p.shift, id = constant(table + (index < p.width ? index : p.width - 1));
                ids[j] = key < len && index < p.width && (unsigned)id < (unsigned)p.num_blocks ? id : -1;
            }
            const auto pick = [&](int j) {
                const int a = j & 1 ? ids[1] : ids[0], b = j & 1 ? ids[3] : ids[2];
                return j & 2 ? b : a;
            };
            const int kid = pick(wk >> 2), vid = pick(lg);
            dead = vid < 0;
            none = !__any(!dead);
            const long long kb = kid < 0 ? 0 : kid, vb = vid < 0 ? 0 : vid;
            k = p.k + kb * p.k_bs + (int64_t)(h * P + (kk & (P - 1))) * W;
            v = p.v + vb * p.v_bs + (int64_t)h * P * W + (vk & (P - 1));
            kf = factor(dead ? 0.f : constant(p.ks + vb * p.ks_bs + h) * p.scale_log2);
            vs = dead ? 0.f : constant(p.vs + vb * p.vs_bs + h);
            blank = vs == 0.f;
            vs = factor(vs);
        }
    }
    // byte offset of key tile 0's row of this lane, and of its row of value column 0
    static __device__ __forceinline__ unsigned key_lane(int W, int lane) {
        const int wk = lane & 15, lg = lane >> 4;
        return (unsigned)(((SMALL ? 0 : 16 * (wk >> 2)) + (wk & 3)) * W + 16 * lg);
    }
    static __device__ __forceinline__ unsigned value_lane(int shift, int lane) {
        return (unsigned)(((lane & 15) << shift) + (SMALL ? 0 : 16 * (lane >> 4)));
    }
};

// Codes are read once, so the row kernel asks for them past the caches' keeping (nontemporal: 108 instead of 123 us for 64 requests of 4600 tokens, 8 heads of
// 128) - where a 128-byte line belongs to one wave's loads.  In blocks of 128 tokens a line of the values holds one column of TWO units, which two waves read:
// it has to stay until the second one comes (142 instead of 126 us otherwise).
template <bool ONCE>
__device__ __forceinline__ u32x4 read_codes(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load((const u32x4*)p);
    else return *(const u32x4*)p;
}

// ---- row kernel ---------------------------------------------------------------------------------------------------------------------------
// (whole: the line is made of row tiles, none of which is cut)
__device__ __forceinline__ long long row_items(const CacheAttnParams& p, const Request& rq, int rows16) {
    const int tiles = (rq.n * p.group + rows16 - 1) / rows16;
    return (long long)tiles * p.Hkv * (p.whole ? 1 : rq.units);
}
__device__ __forceinline__ long long range_of(const CacheAttnParams& p, long long total) {
    const long long per = (total + p.grid - 1) / p.grid;
    return per > p.min_units ? per : p.min_units;
}

// SHIFT: block size, 16 and 32 as one (4), 64 (6), 128 (7)
template <typename T, int W, int NR, int SHIFT>
__global__ __launch_bounds__(256, 2) void cache_rows_kernel(CacheAttnParams p) {
    constexpr bool SMALL = SHIFT < 6;
    using State = RowState<T, W, NR>;
    constexpr int ND = State::ND, NK = W / 64, ROWS = 16 * NR;
    // the next unit's codes are fetched under this one's arithmetic where the registers hold them beside O; else a unit's value columns are
    // taken in parts, as large as the registers hold (width 256, 64 requests of 4096: quarters 172 us, eighths 189; 32 rows of width 128 over 2048: halves 52.5,
    // quarters 58)
    constexpr bool AHEAD = W * NR <= 128;
    constexpr int VN = AHEAD ? ND : W > 192 ? (SMALL ? ND / 8 : ND / 4) : ND / 2;
    __shared__ __align__(8) unsigned short nan_keys[4][4 * W];     // [wave][column][16-key group]
    __shared__ f32x4 join_o[2][NR * ND * 64];
    __shared__ float join_m[4][ROWS], join_l[4][ROWS];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int lg = lane >> 4, wk = lane & 15;
    long long range = 1, start = 0;
    const Place at = find_place(p, [&](const Request& r) { return row_items(p, r, ROWS); },
                                [&](long long total) { range = range_of(p, total); start = range * (long long)blockIdx.x; return start; },
                                blockIdx.x == 0 && wave == 0 ? p.ws_prefix : nullptr);
    if (start >= at.total) return;
    const long long end = start + range < at.total ? start + range : at.total;
    int b = at.b;
    long long off = at.off, cur = start;
    const unsigned key_off = UnitAt<SMALL>::key_lane(W, lane), value_off = UnitAt<SMALL>::value_lane(p.shift, lane);
    State st;
    Request rq = at.rq;
    while (cur < end) {
        const int tiles = (rq.n * p.group + ROWS - 1) / ROWS;
        const int per = p.whole ? 1 : rq.units;            // items of a row tile
        const long long items = (long long)tiles * p.Hkv * per;
        if (off >= items) {                                // (the next request with rows; there is one, cur < end)
            rq = request_of(p, ++b);
            off = 0;
            continue;
        }
        const int ht = (int)(off / per), u0 = (int)(off - (long long)ht * per);
        const int h = ht / tiles, row0 = (ht - h * tiles) * ROWS;
        const int u1 = p.whole || u0 + (end - cur) >= rq.units ? rq.units : (int)(u0 + (end - cur));
        const bool whole = u0 == 0 && u1 == rq.units;
        const int* table = p.tables + (int64_t)b * p.table_stride;
        st.load(p, rq, h, row0, lane);
        st.clear();
        u32x4 kr[4][NK], vr[VN];
        UnitAt<SMALL> here, next;
        const auto load_keys = [&](const UnitAt<SMALL>& a) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < NK; ++i) kr[t][i] = read_codes<true>(a.k + (4 * t * W + 64 * i) + key_off);
        };
        const auto drop_keys = [&]() {                     // (else the last unit's keys stay in registers for a round that never comes)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < NK; ++i) kr[t][i] = __builtin_nondeterministic_value(kr[t][i]);
        };
        const auto load_values = [&](const UnitAt<SMALL>& a, int d0) {
            const int step = fresh_scalar(16 << p.shift);
#pragma unroll
            for (int d = 0; d < VN; ++d) vr[d] = read_codes<SHIFT < 7>(a.v + (d0 + d) * step + value_off);
        };
        int u = u0 + wave;
        if (u < u1) {
            here.find(p, table, rq.len, u, h, W, lane);
            load_keys(here);
            if (AHEAD) load_values(here, 0);
            for (;; u += 4) {
                const bool more = u + 4 < u1;
                if (more) next.find(p, table, rq.len, u + 4, h, W, lane);
                // (a unit without a block is masked altogether: a branch round the arithmetic costs more registers than the kernel has)
                const bool boundary = 64 * u + 64 > st.limit_min || here.none;
                {
                    const int key0 = 64 * u + 16 * lg;
                    f32x4 s[NR][4];
                    typename State::vec8 w[NR][2];
                    st.template scores<true>([&](int t, int c) { return fragment<T>(kr[t][c >> 1][2 * (c & 1)], kr[t][c >> 1][2 * (c & 1) + 1]); }, s);
                    if (!AHEAD) load_values(here, 0);
                    else if (more) load_keys(next);
                    else drop_keys();
                    if (boundary || (SMALL && __any(here.dead))) st.mask(s, key0, here.dead);
                    float top[NR];
                    st.peak(s, here.kf, here.vs, top);
                    st.raise(top);
                    st.weights(s, w, here.kf, here.vs);
                    bool nan = false;
                    const auto part = [&](auto from) {
                        constexpr int D0 = decltype(from)::value;
                        if (64 * u + 64 > rq.len || __any(here.blank)) {
                            const int valid = here.blank ? 0 : rq.len - key0;
#pragma unroll
                            for (int d = 0; d < VN; ++d) vr[d] = clear_behind(vr[d], valid);
                        }
                        if (boundary) {
                            const int slot = fresh_lane(4 * wk + lg);       // the lane's place in nan_keys[wave], 64 apart for each column tile
                            unsigned short* keys = nan_keys[wave] + slot;
                            bool mine = false;
#pragma unroll
                            for (int d = 0; d < VN; ++d) mine |= has_nan(vr[d]);
                            if (!nan && __any(mine)) {
                                nan = true;
                                for (int d = 0; d < ND; ++d) keys[64 * d] = 0;
                            }
                            if (nan) {
#pragma unroll
                                for (int d = 0; d < VN; ++d) {
                                    keys[64 * (D0 + d)] = (unsigned short)take_nan(vr[d]);
                                    __builtin_amdgcn_sched_barrier(0);
                                }
                            }
                        }
                        st.template values<D0, D0 + VN, true>([&](int d, int v) { return fragment<T>(vr[d - D0][2 * v], vr[d - D0][2 * v + 1]); }, w);
                    };
                    fa_static_for<0, ND / VN>([&](auto i) {
                        if constexpr (decltype(i)::value > 0) load_values(here, decltype(i)::value * VN);
                        part(std::integral_constant<int, decltype(i)::value * VN>{});
                    });
                    if (nan) {
                        wave_order();                          // (every lane's marks stand before any lane reads them, and are read before the next unit's)
                        st.note_nan(nan_keys[wave], u, lg);
                        wave_order();
                    }
                }
                if (!more) break;
                if (AHEAD) load_values(next, 0);
                else load_keys(next);
                here = next;
            }
        }
        // the waves' parts joined, the first wave ends with the sums
        const int active = min(4, u1 - u0);
        st.put_nan();
        float sum[NR], top[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) { sum[r] = rows_sum(st.l[r]); top[r] = st.m[r]; }
        if (active > 1) {
            if (lg == 0) {
#pragma unroll
                for (int r = 0; r < NR; ++r) { join_m[wave][16 * r + wk] = top[r]; join_l[wave][16 * r + wk] = sum[r]; }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float all = -INFINITY, total = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) all = __builtin_fmaxf(all, join_m[w][16 * r + wk]);
                const float base = all == -INFINITY ? 0.f : all;
#pragma unroll
                for (int w = 0; w < 4; ++w) total += join_l[w][16 * r + wk] * fast_exp2(join_m[w][16 * r + wk] - base);
                const float f = fast_exp2(top[r] - base);
#pragma unroll
                for (int d = 0; d < ND; ++d) st.o[r][d] *= f;
                top[r] = all;
                sum[r] = total;
            }
#pragma unroll
            for (int step = 2; step >= 1; step >>= 1) {
                if (wave >= step && wave < 2 * step) {
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int d = 0; d < ND; ++d) join_o[wave - step][(r * ND + d) * 64 + lane] = st.o[r][d];
                }
                __syncthreads();
                if (wave < step) {
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int d = 0; d < ND; ++d) st.o[r][d] += join_o[wave][(r * ND + d) * 64 + lane];
                }
                __syncthreads();
            }
        }
        if (wave == 0) {
            if (whole) st.store(p, rq, h, row0, lane, sum);
            else st.park(p, 2ll * blockIdx.x + (cur == start ? 0 : 1), ROWS, 0, lane, sum, top);
        }
        cur += p.whole ? 1 : u1 - u0;
        off += p.whole ? 1 : u1 - u0;
    }
}

// Order of a stretch of MFMAs products, READS operand reads from LDS and vector work: the first reads, then a read for every MFMAS / READS products with VALU vector
// instructions behind each of them.  (Left to itself the compiler waits for every read where it is used and lets the two units take turns.)
template <int MFMAS, int READS, int VALU, int AHEAD>
__device__ __forceinline__ void mix() {
    constexpr int PER = MFMAS / READS;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        if (i + AHEAD < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, VALU, 0);
    }
}

// ---- tile kernel --------------------------------------------------------------------------------------------------------------------------
template <typename T, int W, int NR, bool SMALL>
__global__ __launch_bounds__(256, W > 128 ? 1 : 2) void cache_tile_kernel(CacheAttnParams p) {
    constexpr int ROWS = 64 * NR, NK = W / 64, ND = W / 16, NC = W / 32, KPW = NK, VPW = ND / 4;
    using State = RowState<T, W, NR>;
    using vec8 = typename State::vec8;
    __shared__ u32x4 lds_k[2][4 * NC * 64], lds_v[2][2 * ND * 64];
    __shared__ __align__(8) unsigned short nan_keys[2][4 * W];     // [buffer][column][16-key group]
    __shared__ int nan_found[2];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int lg = lane >> 4, wk = lane & 15;
    // block -> (head, part, tile): the head is the fastest, so that the tiles that share codes run on one XCD where the head count divides 8
    // or is a multiple of it; late tiles (the long ones of a prompt) first.  Where two workgroups per compute unit take all of them, the second ones come in the
    // other order: the longest beside the shortest (one prompt of 2048, 32 / 8 heads of 128:
    // 74.5 -> 70.6 us; eight of 256 over 1024: 53.3 -> 51.6).  `half`: tiles of a head that one workgroup per compute unit takes
    const int idx = (int)blockIdx.x, h = idx % p.Hkv, rest = idx / p.Hkv, part = rest % p.splits, order = rest / p.splits;
    const int half = W <= 128 ? 256 / (p.Hkv * p.splits) : 0x3fffffff;
    long long tile = 0;
    const Place at = find_place(p, [&](const Request& r) { return (long long)((r.n * p.group + ROWS - 1) / ROWS); },
                                [&](long long total) { tile = order >= half && total <= 2 * half ? order - half : total - 1 - order; return tile; },
                                blockIdx.x == 0 && wave == 0 ? p.ws_prefix : nullptr);
    if (order >= at.total || tile >= p.max_tiles) return;      // (more tiles than tokens allow: cu_q is not ascending)
    const Request rq = request_of(p, at.b);
    const int row0 = (int)at.off * ROWS;
    const int* table = p.tables + (int64_t)at.b * p.table_stride;
    State st;
    st.load(p, rq, h, row0 + 16 * NR * wave, lane);
    st.clear();
    const int last = min(row0 + ROWS, rq.n * p.group) - 1;
    const int see = rq.len - rq.n + last / p.group + 1;            // keys that the tile's last row sees
    const int units = see > 0 ? (see + 63) >> 6 : 0;
    const int u0 = (int)((long long)units * part / p.splits), u1 = (int)((long long)units * (part + 1) / p.splits);

    const int tile_min = rq.len - rq.n + row0 / p.group + 1;        // keys that its first row sees
    if (threadIdx.x < 2) nan_found[threadIdx.x] = 0;
    __syncthreads();

    // Operands of a unit: wave w brings key tile w and the value columns of ND / 4 tiles.  The loop runs one unit ahead on the score side: while the
    // matrix pipe forms S(u + 1), the vector unit forms the weights of u; while it adds V(u) P(u), the vector unit looks for the maxima of S(u + 1).  So
    // the keys of u + 2 and the values of u + 1 are fetched in the middle of a round and spread into LDS at its end, two buffers each, one barrier.
    u32x4 kr[KPW], vr[VPW];
    UnitAt<SMALL> here, next, after;
    const unsigned key_off = UnitAt<SMALL>::key_lane(W, lane), value_off = UnitAt<SMALL>::value_lane(p.shift, lane);
    const auto load_keys = [&](const UnitAt<SMALL>& a) {
#pragma unroll
        for (int i = 0; i < KPW; ++i) kr[i] = *(const u32x4*)(a.k + (4 * wave * W + 64 * i) + key_off);
    };
    const auto load_values = [&](const UnitAt<SMALL>& a) {
#pragma unroll
        for (int i = 0; i < VPW; ++i) vr[i] = *(const u32x4*)(a.v + ((16 * (wave * VPW + i)) << p.shift) + value_off);
    };
    const auto spread_keys = [&](int buf) {
#pragma unroll
        for (int i = 0; i < KPW; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                lds_k[buf][(wave * NC + 2 * i + c) * 64 + lane] = __builtin_bit_cast(u32x4, fragment<T>(kr[i][2 * c], kr[i][2 * c + 1]));
    };
    const auto spread_values = [&](const UnitAt<SMALL>& a, int u, int buf) {
        if (64 * u + 64 > rq.len || __any(a.blank)) {
            const int valid = a.blank ? 0 : rq.len - (64 * u + 16 * lg);
#pragma unroll
            for (int i = 0; i < VPW; ++i) vr[i] = clear_behind(vr[i], valid);
        }
        if (64 * u + 64 > tile_min) {                               // (uniform) a unit that some rows see in part
            bool mine = false;
#pragma unroll
            for (int i = 0; i < VPW; ++i) {
                mine |= has_nan(vr[i]);
                nan_keys[buf][64 * (wave * VPW + i) + 4 * wk + lg] = (unsigned short)take_nan(vr[i]);
            }
            if (mine) nan_found[buf] = u + 1;                       // (no other value is written here: a unit's mark is its own number)
        }
#pragma unroll
        for (int i = 0; i < VPW; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                lds_v[buf][((wave * VPW + i) * 2 + c) * 64 + lane] = __builtin_bit_cast(u32x4, fragment<T>(vr[i][2 * c], vr[i][2 * c + 1]));
    };
    f32x4 s[2][NR][4];
    const auto scores = [&](int buf, f32x4 (&to)[NR][4]) {
        st.template scores<false>([&](int t, int c) { return __builtin_bit_cast(vec8, lds_k[buf][(t * NC + c) * 64 + lane]); }, to);
    };
    // what stands between a unit's scores and its weights
    const auto prepare = [&](int u, const UnitAt<SMALL>& a, f32x4 (&x)[NR][4], float (&top)[NR]) {
        if (64 * u + 64 > st.limit_min || __any(a.dead)) st.mask(x, 64 * u + 16 * lg, a.dead);
        st.peak(x, a.kf, a.vs, top);
    };
    if (u0 < u1) {
        here.find(p, table, rq.len, u0, h, W, lane);
        load_keys(here);
        load_values(here);
        spread_keys(0);
        spread_values(here, u0, 0);
        next.find(p, table, rq.len, min(u0 + 1, u1 - 1), h, W, lane);
        load_keys(next);
        spread_keys(1);
    }
    __syncthreads();
    if (u0 < u1) {
        float top[NR];
        scores(0, s[0]);
        prepare(u0, here, s[0], top);
        st.raise(top);
    }
    __syncthreads();                                                // (unit u0's keys are read: round u0 fetches u0 + 2's over them)
    const auto round = [&](int u, auto which) {
        constexpr int A = decltype(which)::value, B = A ^ 1;        // buffers and scores of this unit and of the next
        const bool more = u + 1 < u1;
        // (behind the end everything goes on with the last unit's operands, and is dropped: a branch round the fetches costs more registers than there are)
        if (!SMALL) after.find(p, table, rq.len, min(u + 2, u1 - 1), h, W, lane);
        vec8 w[NR][2];
        __builtin_amdgcn_sched_barrier(0);
        scores(B, s[B]);
        st.weights(s[A], w, here.kf, here.vs);
        mix<4 * NC * NR, 4 * NC, 8, 2>();
        __builtin_amdgcn_sched_barrier(0);
        if (SMALL) after.find(p, table, rq.len, min(u + 2, u1 - 1), h, W, fresh_lane(lane));     // (addresses of every lane: formed where registers are free)
        load_keys(after);                                           // (here, where the scores of u have left their registers)
        load_values(next);
        float top[NR];
        if (64 * u + 128 > st.limit_min || __any(next.dead)) st.mask(s[B], 64 * u + 64 + 16 * lg, next.dead);
        __builtin_amdgcn_sched_barrier(0);
        st.template values<0, ND, false>([&](int d, int v) { return __builtin_bit_cast(vec8, lds_v[A][(d * 2 + v) * 64 + lane]); }, w);
        st.peak(s[B], next.kf, next.vs, top);
        mix<2 * ND * NR, 2 * ND, 1, SMALL ? 2 : 4>();
        __builtin_amdgcn_sched_barrier(0);
        if (nan_found[A] == u + 1) st.note_nan(nan_keys[A], u, lg);
        if (more) st.raise(top);
        spread_values(next, u + 1, B);
        spread_keys(A);
        here = next;
        next = after;
        __syncthreads();
    };
    for (int u = u0; u < u1; u += 2) {
        round(u, std::integral_constant<int, 0>{});
        if (u + 1 < u1) round(u + 1, std::integral_constant<int, 1>{});
    }
    st.put_nan();
    float sum[NR], top[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) { sum[r] = rows_sum(st.l[r]); top[r] = st.m[r]; }
    if (p.splits == 1) st.store(p, rq, h, row0 + 16 * NR * wave, lane, sum);
    else st.park(p, ((long long)h * p.max_tiles + tile) * p.splits + part, ROWS, 16 * NR * wave, lane, sum, top);
}

// ---- join kernel: partial sums of join_rows rows of one (request, key/value head, row tile), 64 columns per workgroup --------------------------
// Bound: latency, of which the loads of a strand of slots are most; so few rows are spread over more workgroups of more strands, and a strand has
// four slots' loads in flight.  The order of the sums is fixed by the layout: results are the same from call to call.
template <typename T, bool TILE>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttnParams p, int W, int rows16) {
    constexpr int DEEP = 4;
    __shared__ f32x4 part_o[256];
    __shared__ float part_m[256], part_l[256];
    int b, h, tile;
    long long item0 = 0, range = 1, w0, w1, slot0 = 0;
    if constexpr (TILE) {
        h = (int)blockIdx.x % p.Hkv;
        const long long t = (int)blockIdx.x / p.Hkv;
        if (t >= p.ws_prefix[p.B] || t >= p.max_tiles) return;
        int lo = 0, hi = p.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.ws_prefix[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        tile = (int)(t - p.ws_prefix[b]);
        w0 = 0;
        w1 = p.splits - 1;
        slot0 = ((long long)h * p.max_tiles + t) * p.splits;
    } else {
        b = (int)blockIdx.x / p.Hkv;
        h = (int)blockIdx.x - b * p.Hkv;
        tile = (int)blockIdx.y / p.join_chunks;
    }
    const int chunk = (int)blockIdx.y % p.join_chunks, tiles_y = (int)gridDim.y / p.join_chunks;
    const Request rq = request_of(p, b);
    const int rows = rq.n * p.group, tiles = (rows + rows16 - 1) / rows16, tid = (int)threadIdx.x;
    for (; tile < tiles; tile += TILE ? tiles : tiles_y) {      // (more rows than the grid was told: every one is still reached)
        if constexpr (!TILE) {
            range = range_of(p, p.ws_prefix[p.B]);
            item0 = p.ws_prefix[b] + ((long long)h * tiles + tile) * rq.units;
            w0 = item0 / range;
            w1 = (item0 + rq.units - 1) / range;
            if (w0 == w1) continue;                                    // (finished by one workgroup)
        }
        // threads: strands of slots x rows x 16 groups of four columns
        const int there = min(rows16, rows - tile * rows16);
        for (int base = chunk * p.join_rows; base < there; base += p.join_chunks * p.join_rows) {
            const int live = min(p.join_rows, there - base);
            const int lanes = live > 8 ? 256 : live > 4 ? 128 : live > 2 ? 64 : live > 1 ? 32 : 16;
            const int strands = 256 / lanes, strand = tid / lanes, row = (tid % lanes) >> 4, c = tid & 15;
            const int col = 64 * (int)blockIdx.z + 4 * c;
            float top = -INFINITY, sum = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            if (row < live) {
                for (long long w = w0 + strand; w <= w1; w += DEEP * strands) {
                    f32x2c ml[DEEP];
                    f32x4 v[DEEP];
#pragma unroll
                    for (int j = 0; j < DEEP; ++j) {
                        const long long wj = w + j * strands <= w1 ? w + j * strands : w;
                        const long long slot = TILE ? slot0 + wj : 2 * wj + (wj * range >= item0 ? 0 : 1);
                        const long long at = slot * rows16 + base + row;
                        ml[j] = *(const f32x2c*)(p.ws_ml + 2 * at);
                        v[j] = *(const f32x4*)(p.ws_o + at * W + col);
                    }
#pragma unroll
                    for (int j = 0; j < DEEP; ++j) {
                        if (w + j * strands > w1) continue;
                        const float m = ml[j][0], now = __builtin_fmaxf(top, m), b0 = now == -INFINITY ? 0.f : now;
                        const float f0 = fast_exp2(top - b0), f1 = fast_exp2(m - b0);
                        o = o * f0 + v[j] * f1;
                        sum = sum * f0 + ml[j][1] * f1;
                        top = now;
                    }
                }
            }
            part_o[tid] = o;
            part_m[tid] = top;
            part_l[tid] = sum;
            __syncthreads();
            if (strand == 0 && row < live) {
                for (int s = 1; s < strands; ++s) {
                    const int i = s * lanes + tid;
                    const float m = part_m[i], now = __builtin_fmaxf(top, m), b0 = now == -INFINITY ? 0.f : now;
                    const float f0 = fast_exp2(top - b0), f1 = fast_exp2(m - b0);
                    o = o * f0 + part_o[i] * f1;
                    sum = sum * f0 + part_l[i] * f1;
                    top = now;
                }
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                const int r = tile * rows16 + base + row, i = r / p.group, g = r - i * p.group;
                if (col < p.D) {
                    o *= inv;
                    T* dst = (T*)p.o + (int64_t)(rq.first + i) * p.o_st + (int64_t)(h * p.group + g) * p.o_sh + col;
                    *(u32x2c*)dst = u32x2c{pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3])};
                }
            }
            __syncthreads();
        }
    }
}

template <typename T, int W, int NR>
const void* rows_kernel(int shift) {
    return shift < 6 ? (const void*)cache_rows_kernel<T, W, NR, 4> : shift == 6 ? (const void*)cache_rows_kernel<T, W, NR, 6> : (const void*)cache_rows_kernel<T, W, NR, 7>;
}
template <typename T, int W>
hipError_t launch_width(const CacheAttnParams& p, const CacheAttnPlan& plan, hipStream_t stream) {
    const bool small = p.shift < 6;
    const void* k;
    if (plan.tile) k = plan.nr == 1 ? (small ? (const void*)cache_tile_kernel<T, W, 1, true> : (const void*)cache_tile_kernel<T, W, 1, false>)
                                    : (small ? (const void*)cache_tile_kernel<T, W, 2, true> : (const void*)cache_tile_kernel<T, W, 2, false>);
    else k = plan.nr == 1 || W > 128 ? rows_kernel<T, W, 1>(p.shift) : rows_kernel<T, (W <= 128 ? W : 128), 2>(p.shift);
    return launch1(k, dim3((unsigned)plan.grid), dim3(256), 0, stream, p);
}
template <typename T>
hipError_t launch_typed(const CacheAttnParams& p, const CacheAttnPlan& plan, hipStream_t stream) {
    hipError_t e = plan.width == 64 ? launch_width<T, 64>(p, plan, stream) : plan.width == 128 ? launch_width<T, 128>(p, plan, stream)
                 : plan.width == 192 ? launch_width<T, 192>(p, plan, stream) : launch_width<T, 256>(p, plan, stream);
    if (e != hipSuccess || (plan.tile ? plan.splits == 1 : p.whole)) return e;
    const int rows16 = (plan.tile ? 64 : 16) * plan.nr;
    CacheAttnParams arg = p;
    int W = plan.width, rows = rows16;
    void* args[] = {&arg, &W, &rows};
    const dim3 grid((unsigned)(p.Hkv * (plan.tile ? plan.max_tiles : p.B)), (unsigned)(p.join_chunks * (plan.tile ? 1 : plan.max_tiles)), (unsigned)(plan.width / 64));
    return hipLaunchKernel(plan.tile ? (const void*)cache_join_kernel<T, true> : (const void*)cache_join_kernel<T, false>, grid, dim3(256), args, 0, stream);
}

}  // namespace

hipError_t launch_cache_attn(const CacheAttnParams& p, const CacheAttnPlan& plan, int dtype, hipStream_t stream) {
    return dtype == 0 ? launch_typed<_Float16>(p, plan, stream) : launch_typed<__bf16>(p, plan, stream);
}

}  // namespace fa
