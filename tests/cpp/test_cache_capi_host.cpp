// Host-only sanitizer run of csrc/fa_cache_capi.cpp: every refusal, plan invariants over a grid of requests, extreme sizes.  The kernels are replaced
// by launchers that check what they were handed; no pointer is followed.
#include "flash_attention_amd.h"
#include "fa_cache.h"

#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int g_launches = 0;
static fa::CacheAttnParams g_attn;
static fa::CacheAttnPlan g_plan;
static fa::RopeParams g_rope;
static fa::AppendParams g_append;
static bool g_vec;
static int g_hc;

namespace fa {
hipError_t launch_rope_fwd(const RopeParams& p, int, bool vec, int hc, bool, hipStream_t) { ++g_launches; g_rope = p; g_vec = vec; g_hc = hc; return hipSuccess; }
hipError_t launch_rope_bwd(const RopeParams& p, int, bool vec, int hc, bool, hipStream_t) { ++g_launches; g_rope = p; g_vec = vec; g_hc = hc; return hipSuccess; }
hipError_t launch_cache_tables(const TablesParams&, hipStream_t) { ++g_launches; return hipSuccess; }
hipError_t launch_cache_append(const AppendParams& p, int, hipStream_t) { ++g_launches; g_append = p; return hipSuccess; }
hipError_t launch_cache_attn(const CacheAttnParams& p, const CacheAttnPlan& plan, int, hipStream_t) { ++g_launches; g_attn = p; g_plan = plan; return hipSuccess; }
}  // namespace fa

#define CHECK(x) do { if (!(x)) { printf("FAILED %s:%d: %s (%s)\n", __FILE__, __LINE__, #x, fa_last_error()); exit(1); } } while (0)

static char buf[1 << 16] __attribute__((aligned(64)));

static int rope(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t D, int64_t R, int dtype, int wdtype, float eps, int inter, int pos_bytes, const int64_t* st, const void* q,
                const void* table, bool bwd, int64_t ws) {
    int64_t s[6][3];
    for (int i = 0; i < 6; ++i) for (int j = 0; j < 3; ++j) s[i][j] = st[j];
    const float* t = (const float*)table;
    if (bwd) return fa_qk_norm_rope_bwd(q, buf, buf, buf, buf, buf, buf, buf, buf, buf, wdtype, ws ? buf : nullptr, ws, t, 100, buf, pos_bytes, 0, B, L, H, Hk, D, R, s, dtype, eps, inter, nullptr);
    return fa_qk_norm_rope_fwd(q, buf, buf, buf, buf, buf, wdtype, t, 100, buf, pos_bytes, 0, B, L, H, Hk, D, R, s, dtype, eps, inter, nullptr);
}

int main() {
    const int64_t st[3] = {1 << 20, 64, 4096};
    // ---- rotation
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_OK && g_vec);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 2, 1e-6f, 1, 8, st, buf + 2, buf, false, 0) == FA_OK && !g_vec);      // unaligned: one element at a time
    CHECK(rope(2, 8, 4, 2, 80, 64, 1, 2, 1e-6f, 1, 8, st, buf, buf, false, 0) == FA_OK && !g_vec);
    CHECK(rope(2, 8, 4, 2, 64, 0, 1, 2, 0.f, 0, 8, st, buf, nullptr, false, 0) == FA_OK);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf + 1, buf, false, 0) == FA_ERR_MISALIGNED);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, nullptr, buf, false, 0) == FA_ERR_NULL_POINTER);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, nullptr, false, 0) == FA_ERR_NULL_POINTER);
    CHECK(rope(0, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SHAPE);
    CHECK(rope(2, 8, 4, 2, 63, 62, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SHAPE);
    CHECK(rope(2, 8, 4, 2, 514, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SHAPE);
    CHECK(rope(2, 8, 4, 2, 64, 66, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SHAPE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 3, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_DTYPE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 0, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_DTYPE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 2, st, buf, buf, false, 0) == FA_ERR_BAD_DTYPE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, -1.f, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SCALE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, NAN, 0, 4, st, buf, buf, false, 0) == FA_ERR_BAD_SCALE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 2, 4, st, buf, buf, false, 0) == FA_ERR_BAD_OPTION);
    CHECK(rope(1 << 20, 1 << 20, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_TOO_LARGE);
    CHECK(rope(1ll << 62, 1ll << 62, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, false, 0) == FA_ERR_TOO_LARGE);
    const int64_t bad_st[3] = {-1, 64, 64}, far_st[3] = {1ll << 50, 64, 64};
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, bad_st, buf, buf, false, 0) == FA_ERR_BAD_STRIDE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, far_st, buf, buf, false, 0) == FA_ERR_BAD_STRIDE);
    const int64_t need = fa_qk_norm_rope_workspace(2, 8, 4, 2, 64);
    CHECK(need > 0 && rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, true, need) == FA_OK);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, true, need - 1) == FA_ERR_WORKSPACE);
    CHECK(rope(2, 8, 4, 2, 64, 64, 1, 1, 1e-6f, 0, 4, st, buf, buf, true, 0) == FA_ERR_NULL_POINTER);
    // every launch covers its items, and partial weight gradients fit the workspace
    for (int64_t B : {1, 3, 700}) for (int64_t L : {1, 7, 4096}) for (int64_t H : {1, 5, 32}) for (int64_t D : {32, 64, 80, 128, 256, 512}) for (int bwd = 0; bwd < 2; ++bwd) {
        CHECK(rope(B, L, H, 2, D, 32, 1, 1, 1e-6f, 0, 4, st, buf, buf, bwd, bwd ? fa_qk_norm_rope_workspace(B, L, H, 2, D) : 0) == FA_OK);
        for (int i = 0; i < 2; ++i) {
            const fa::RopeSide& s = g_rope.side[i];
            CHECK((int64_t)s.chunks * g_hc >= s.heads && (int64_t)(s.chunks - 1) * g_hc < s.heads && s.items == B * L * s.chunks && s.blocks >= 1);
            if (bwd) CHECK((char*)(s.dw_part + (int64_t)s.blocks * D) <= buf + fa_qk_norm_rope_workspace(B, L, H, 2, D));
            else CHECK(s.blocks >= 2048 /* the kernels stride over more */ || (int64_t)s.blocks * 256 >= (int64_t)s.items * (g_vec ? D * 2 / 32 : 64));
        }
    }
    // ---- tables
    int32_t* ip = (int32_t*)buf;
    const auto tables = [&](int64_t B, int64_t T, int64_t P, int64_t width, int64_t stride, int64_t pool, int32_t* seq) {
        return fa_cache_tables(seq, ip, ip, stride, width, ip, pool, ip, B, T, P, ip, ip, ip, ip, T ? ip : nullptr, T ? ip : nullptr, nullptr);
    };
    CHECK(tables(4, 10, 16, 8, 8, 100, ip) == FA_OK && tables(4, 0, 16, 8, 8, 100, ip) == FA_OK);
    CHECK(tables(4, 10, 16, 8, 8, 100, nullptr) == FA_ERR_NULL_POINTER);
    CHECK(tables(4, 10, 17, 8, 8, 100, ip) == FA_ERR_BAD_SHAPE && tables(0, 10, 16, 8, 8, 100, ip) == FA_ERR_BAD_SHAPE && tables(4, -1, 16, 8, 8, 100, ip) == FA_ERR_BAD_SHAPE);
    CHECK(tables(4, 10, 16, 8, 7, 100, ip) == FA_ERR_BAD_STRIDE);
    CHECK(tables(4, 10, 128, 8, 8, 1 << 30, ip) == FA_ERR_TOO_LARGE && tables(4, 10, 128, 1 << 25, 1 << 25, 100, ip) == FA_ERR_TOO_LARGE && tables(1ll << 40, 10, 16, 8, 8, 100, ip) == FA_ERR_TOO_LARGE);
    // ---- append
    const auto append = [&](int64_t T, int64_t H, int64_t D, int64_t W, int64_t N, int64_t P, int64_t ts, int64_t bs, int64_t ss, int dtype, char* k) {
        const int64_t t4[4] = {ts, D, ts, D}, b4[4] = {bs, bs, ss, ss};
        return fa_cache_append(k, buf, ip, buf, buf, (float*)buf, (float*)buf, T, H, D, W, N, P, t4, b4, dtype, nullptr);
    };
    CHECK(append(5, 2, 64, 64, 4, 16, 128, 2 * 16 * 64, 2, 1, buf) == FA_OK);
    const int before = g_launches;
    CHECK(append(0, 2, 64, 64, 4, 16, 128, 2 * 16 * 64, 2, 1, buf) == FA_OK && g_launches == before);
    CHECK(append(5, 2, 64, 64, 4, 16, 128, 2 * 16 * 64, 2, 2, buf) == FA_ERR_BAD_DTYPE);
    CHECK(append(5, 2, 64, 128, 4, 16, 128, 2 * 16 * 64, 2, 1, buf) == FA_ERR_BAD_SHAPE && append(5, 2, 60, 64, 4, 16, 128, 2048, 2, 1, buf) == FA_ERR_BAD_SHAPE);
    CHECK(append(5, 2, 264, 320, 4, 16, 128, 1 << 20, 2, 1, buf) == FA_ERR_BAD_SHAPE && append(5, 0, 64, 64, 4, 16, 128, 2048, 2, 1, buf) == FA_ERR_BAD_SHAPE);
    CHECK(append(5, 2, 64, 64, 4, 16, 128, 2 * 16 * 64 - 16, 2, 1, buf) == FA_ERR_BAD_STRIDE && append(5, 2, 64, 64, 4, 16, 128, 2 * 16 * 64 + 8, 2, 1, buf) == FA_ERR_BAD_STRIDE);
    CHECK(append(5, 2, 64, 64, 4, 16, 128, 2048, 1, 1, buf) == FA_ERR_BAD_STRIDE);
    CHECK(append(5, 2, 64, 64, 4, 16, 132, 2048, 2, 1, buf) == FA_ERR_MISALIGNED && append(5, 2, 64, 64, 4, 16, 128, 2048, 2, 1, buf + 8) == FA_ERR_MISALIGNED);
    CHECK(append(5, 2, 64, 64, 1ll << 40, 16, 128, 2048, 2, 1, buf) == FA_ERR_TOO_LARGE && append(1ll << 40, 2, 64, 64, 4, 16, 128, 2048, 2, 1, buf) == FA_ERR_TOO_LARGE);
    for (int64_t T : {1, 64, 5000, 1 << 20}) {
        CHECK(append(T, 8, 128, 128, 4, 64, 1024, 8 * 64 * 128, 8, 0, buf) == FA_OK);
        CHECK(g_append.window >= 4 && g_append.window <= 64 && (g_append.window & (g_append.window - 1)) == 0);
    }
    // ---- attention
    const auto attn = [&](int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t N, int64_t P, int64_t width, int64_t most, float scale, int64_t short_by, int dtype) {
        const int64_t W = (D + 63) / 64 * 64, t4[4] = {H * D, D, H * D, D}, bs = Hk * P * W, b4[4] = {bs, bs, Hk, Hk};
        const int64_t ws = fa_cache_attn_workspace(B, T, H, Hk, D, P, width, most);
        if (ws < 0) return (int)ws;
        return fa_cache_attn(buf, buf, buf, buf, (float*)buf, (float*)buf, ip, ip, ip, buf, ws - short_by, B, T, H, Hk, D, W, N, P, width, width, most, t4, b4, dtype, scale, nullptr);
    };
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_OK);
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 500, 1, 0.1f, 1, 1) == FA_ERR_WORKSPACE && attn(2, 2, 8, 2, 128, 10, 64, 500, 1, 0.1f, 0, 1) == FA_OK);
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 2) == FA_ERR_BAD_DTYPE);
    CHECK(attn(2, 2, 8, 3, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE && attn(2, 2, 8, 2, 130, 10, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE);
    CHECK(attn(2, 2, 8, 2, 128, 10, 48, 5, 1, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE && attn(0, 2, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE);
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 5, 0, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE && attn(2, 2, 8, 2, 128, 0, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_BAD_SHAPE);
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 5, 1, 0.f, 0, 1) == FA_ERR_BAD_SCALE && attn(2, 2, 8, 2, 128, 10, 64, 5, 1, INFINITY, 0, 1) == FA_ERR_BAD_SCALE);
    CHECK(attn(2, 1ll << 40, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_TOO_LARGE && attn(1ll << 40, 2, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_ERR_TOO_LARGE);
    CHECK(attn(2, 2, 8, 2, 128, 10, 64, 1ll << 40, 1, 0.1f, 0, 1) == FA_ERR_TOO_LARGE);
    const int l0 = g_launches;
    CHECK(attn(2, 0, 8, 2, 128, 10, 64, 5, 1, 0.1f, 0, 1) == FA_OK && g_launches == l0);
    // plans: the workspace holds every slot that the kernels address, grids cover what they have to
    for (int64_t B : {1, 2, 64, 5000}) for (int64_t T : {1, 7, 64, 4096}) for (int64_t Hk : {1, 8}) for (int64_t group : {1, 4, 16, 48}) for (int64_t D : {8, 64, 128, 192, 256})
        for (int64_t width : {1, 17, 4096}) for (int64_t most : {1, 2, 9, 1000}) {
            CHECK(attn(B, T, Hk * group, Hk, D, 10, 64, width, most, 0.1f, 0, 1) == FA_OK);
            const int64_t W = (D + 63) / 64 * 64;
            CHECK(g_plan.width == W && g_plan.grid >= 1 && g_attn.grid == g_plan.grid && (g_plan.ws_ml & 15) == 0 && (g_plan.ws_prefix & 7) == 0);
            const bool joined = g_plan.tile ? g_plan.splits > 1 : !g_plan.whole;
            CHECK(joined ? g_plan.ws_prefix + 8 * (B + 1) <= g_plan.bytes : !g_attn.ws_o && !g_attn.ws_ml && !g_attn.ws_prefix);
            int64_t slots, rows;
            if (g_plan.tile) {
                rows = 64 * g_plan.nr;
                slots = joined ? Hk * g_plan.max_tiles * g_plan.splits : 0;
                CHECK(g_plan.grid == Hk * g_plan.max_tiles * g_plan.splits && g_plan.max_tiles >= (T * group + rows - 1) / rows);
            } else {
                rows = 16 * g_plan.nr;
                slots = !joined ? 0 : 2ll * g_plan.grid;
                CHECK(g_plan.nr == 1 || W <= 128);
            }
            CHECK(g_plan.ws_ml - g_plan.ws_o >= slots * rows * W * 4 && g_plan.ws_prefix - g_plan.ws_ml >= slots * rows * 8);
        }
    printf("PASSED (%d launches)\n", g_launches);
    return 0;
}
