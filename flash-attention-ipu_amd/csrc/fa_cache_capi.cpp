// C entry points of the operators around attention over an 8-bit key/value cache (include/flash_attention_amd.h): validate, choose the
// launch, enqueue on the caller's stream.  No allocation, no synchronisation, no exceptions.
#include "flash_attention_amd.h"

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "fa_cache.h"

namespace {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
    char text[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return fa::set_error(code, text);
}
int launched(hipError_t e) { return e == hipSuccess ? FA_OK : fail(FA_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e)); }

constexpr int64_t kMaxCount = 1ll << 30;      // rows, items, tokens: 32-bit indexes with room for a grid's stride
constexpr int64_t kMaxGrid = 1ll << 23;       // workgroups along x: times 256 threads stays below 2^32
constexpr int64_t kMaxStride = 1ll << 40;     // elements: products with 32-bit indexes stay inside 64 bits
constexpr int kCus = 256;                     // compute units of an MI355X: sizes grids, never correctness

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// ---- norm and rotation ------------------------------------------------------------------------------------------------------------------
// Workgroups per side.  Backward: also the rows of partial weight gradients.  16384 tokens of 32 + 8 heads of 128 in bf16: 138 us with 256, 100 with 512, 101 with
// 768, 105 with 1024; 2048 tokens 22.5, 20.7, 22.3, 24.9.  Forward: flat between 1024 and 4096 (59 .. 61 us; 512: 66).
constexpr int kRopeMaxBlocks = 768;
constexpr int kRopeFwdBlocks = 2048;

struct RopeCall {
    fa::RopeParams p;
    bool vec, stream_past;
    int hc, es;
};

int rope_common(RopeCall* c, const void* q_weight, const void* k_weight, int32_t weight_dtype, const float* table, int64_t table_rows, const void* positions,
                int32_t position_bytes, int64_t position_stride, int64_t B, int64_t L, int64_t heads, int64_t heads_kv, int64_t D, int64_t R,
                const int64_t (*strides)[3], int n_strides, int32_t dtype, float eps, int32_t interleaved) {
    if (B < 1 || L < 1 || heads < 1 || heads_kv < 1) return fail(FA_ERR_BAD_SHAPE, "batch, length, heads and heads_kv must be >= 1");
    if (D < 2 || D > 512 || D % 2) return fail(FA_ERR_BAD_SHAPE, "head dim must be even and 2 .. 512 (got %lld)", (long long)D);
    if (R < 0 || R > D || R % 2) return fail(FA_ERR_BAD_SHAPE, "rotary dim must be even and 0 .. head dim (got %lld)", (long long)R);
    if (dtype < 0 || dtype > 2) return fail(FA_ERR_BAD_DTYPE, "dtype must be FA_DTYPE_F16/BF16/F32 (got %d)", dtype);
    if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != FA_DTYPE_F32)
        return fail(FA_ERR_BAD_DTYPE, "weights must have the operands' dtype or FA_DTYPE_F32 (got %d)", weight_dtype);
    if (R > 0 && (!table || table_rows < 1)) return fail(FA_ERR_NULL_POINTER, "a rotation needs a table of cosines and sines");
    if (positions && position_bytes != 4 && position_bytes != 8) return fail(FA_ERR_BAD_DTYPE, "positions must be 4- or 8-byte integers (got %d)", position_bytes);
    if (positions && (position_stride < 0 || position_stride >= kMaxStride)) return fail(FA_ERR_BAD_STRIDE, "bad position stride");
    if (!(eps >= 0.f) || !isfinite(eps)) return fail(FA_ERR_BAD_SCALE, "eps must be finite and >= 0 (got %g)", (double)eps);
    if (!(interleaved == 0 || interleaved == 1)) return fail(FA_ERR_BAD_OPTION, "interleaved must be 0 or 1 (got %d)", interleaved);
    if (B > kMaxCount || L > kMaxCount || heads > kMaxCount || heads_kv > kMaxCount || table_rows > (1ll << 40)) return fail(FA_ERR_TOO_LARGE, "sizes must be <= 2^30");
    if (B * L > kMaxCount || B * L * (heads > heads_kv ? heads : heads_kv) > kMaxCount) return fail(FA_ERR_TOO_LARGE, "more than 2^30 rows of queries or keys");
    const int es = dtype == FA_DTYPE_F32 ? 4 : 2;
    bool wide = (D == 32 || D == 64 || D == 128 || D == 256) && R % 16 == 0;
    for (int i = 0; i < n_strides; ++i)
        for (int j = 0; j < 3; ++j) {
            if (strides[i][j] < 0 || strides[i][j] >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "stride %lld is negative or too large", (long long)strides[i][j]);
            if (strides[i][j] % (16 / es)) wide = false;
        }
    fa::RopeParams& p = c->p;
    p = fa::RopeParams{};
    p.table = table; p.table_rows = R > 0 ? table_rows : (1ll << 62); p.positions = positions; p.pos64 = position_bytes == 8; p.pos_sb = position_stride;
    p.L = (int32_t)L; p.D = (int32_t)D; p.R = (int32_t)R; p.interleaved = interleaved; p.w_f32 = weight_dtype == FA_DTYPE_F32; p.eps = eps;
    p.side[0].w = q_weight; p.side[1].w = k_weight;
    p.side[0].heads = (int32_t)heads; p.side[1].heads = (int32_t)heads_kv;
    if (!aligned(table, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16)) wide = false;
    c->vec = wide;
    c->es = es;
    return FA_OK;
}

// Heads per lane group, items and workgroups of both sides.  What moves more than the 256 MB of the last cache is read and written past it (16384 tokens of
// 32 + 8 heads of 128 in bf16: forward 65.2 -> 60.4 us, backward 105 -> 100; 8192 tokens, 168 and 252 MB, lose by it: 30.3 -> 32.7 and 51.3 -> 55.4).  Two heads
// per lane group fetch cosines, sines and position once and keep more loads in flight: 68.8 -> 60.3 us there, 62.3 -> 57.4 for 8192 tokens of 32-bit rows and
// 10.5 -> 9.5 for 1024; 16-bit rows inside the cache want the lanes instead (4096 tokens: 17.8 us with one, 19.5 with two).  Four heads: 62.7.
void rope_shape(RopeCall* c, int64_t B, bool backward) {
    fa::RopeParams& p = c->p;
    const int lpr = c->vec ? p.D * c->es / 32 : 64;
    const int64_t tokens = B * p.L, rows = tokens * (p.side[0].heads + p.side[1].heads);
    c->stream_past = rows * p.D * c->es * (backward ? 3 : 2) > (256ll << 20);
    c->hc = c->vec && (c->es == 4 || c->stream_past) ? 2 : 1;
    for (fa::RopeSide& s : p.side) {
        s.chunks = (int32_t)up(s.heads, c->hc);
        s.items = (int32_t)(tokens * s.chunks);
        int64_t blocks = up((int64_t)s.items * lpr, 256);
        if (backward && blocks > kRopeMaxBlocks) blocks = kRopeMaxBlocks;
        if (blocks > kRopeFwdBlocks) blocks = kRopeFwdBlocks;          // (the kernels stride over what is left)
        s.blocks = (int32_t)blocks;
        s.head_inner = s.x_sh <= s.x_sl;
    }
}

// ---- cache ------------------------------------------------------------------------------------------------------------------------------
int block_shift(int64_t P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : -1; }

int cache_geometry(int64_t num_blocks, int64_t heads_kv, int64_t block_size, int64_t D, int64_t W, const int64_t* strides4, const void* k, const void* v) {
    if (block_shift(block_size) < 0) return fail(FA_ERR_BAD_SHAPE, "block size must be 16, 32, 64 or 128 (got %lld)", (long long)block_size);
    if (D < 8 || D > 256 || D % 8) return fail(FA_ERR_BAD_SHAPE, "head dim must be a multiple of 8 up to 256 (got %lld)", (long long)D);
    if (W != up(D, 64) * 64) return fail(FA_ERR_BAD_SHAPE, "cache width must be the head dim rounded up to a multiple of 64 (got %lld for head dim %lld)", (long long)W, (long long)D);
    if (num_blocks < 1 || heads_kv < 1) return fail(FA_ERR_BAD_SHAPE, "num_blocks and heads_kv must be >= 1");
    if (num_blocks * block_size > 0x7fffffffll || num_blocks > kMaxCount) return fail(FA_ERR_TOO_LARGE, "more than 2^31 - 1 slots");
    if (heads_kv > 32767 || heads_kv * block_size * W > 0x3fffffffll) return fail(FA_ERR_TOO_LARGE, "a block holds more than 2^30 bytes");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(FA_ERR_MISALIGNED, "caches must be 16-byte aligned");
    for (int i = 0; i < 2; ++i)
        if (strides4[i] % 16 || strides4[i] < heads_kv * block_size * W || strides4[i] >= kMaxStride)
            return fail(FA_ERR_BAD_STRIDE, "block stride must be a multiple of 16 bytes and hold a block (got %lld)", (long long)strides4[i]);
    for (int i = 2; i < 4; ++i)
        if (strides4[i] < heads_kv || strides4[i] >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "scale stride must hold a block's heads (got %lld)", (long long)strides4[i]);
    return FA_OK;
}

int attn_plan(int64_t B, int64_t T, int64_t heads, int64_t heads_kv, int64_t D, int64_t block_size, int64_t max_blocks, int64_t max_q_len, fa::CacheAttnPlan* out) {
    if (B < 1 || T < 0 || heads < 1 || heads_kv < 1 || max_blocks < 1) return fail(FA_ERR_BAD_SHAPE, "requests, heads and table width must be >= 1, tokens >= 0");
    if (heads % heads_kv) return fail(FA_ERR_BAD_SHAPE, "heads must be a multiple of heads_kv (got %lld, %lld)", (long long)heads, (long long)heads_kv);
    if (D < 8 || D > 256 || D % 8) return fail(FA_ERR_BAD_SHAPE, "head dim must be a multiple of 8 up to 256 (got %lld)", (long long)D);
    if (block_shift(block_size) < 0) return fail(FA_ERR_BAD_SHAPE, "block size must be 16, 32, 64 or 128 (got %lld)", (long long)block_size);
    if (max_q_len < 1) return fail(FA_ERR_BAD_SHAPE, "max_q_len must be >= 1");
    if (B > (1 << 24) || T > kMaxCount || heads > 32767 || T * heads > kMaxCount) return fail(FA_ERR_TOO_LARGE, "more than 2^24 requests or 2^30 query rows");
    if (max_blocks > kMaxCount || max_blocks * block_size > 0x7fffffffll) return fail(FA_ERR_TOO_LARGE, "a table row addresses more than 2^31 - 1 tokens");
    fa::CacheAttnPlan p{};
    const int64_t group = heads / heads_kv, W = up(D, 64) * 64;
    if (max_q_len > T) max_q_len = T > 0 ? T : 1;
    const int64_t rows = max_q_len * group, max_units = up(max_blocks * block_size, 64);
    p.width = (int32_t)W;
    // The row kernel reads the cache once per row tile: 32 rows, 16 above width 128.  64 requests of 2048 tokens, 8 heads, row kernel against tile kernel: width 64:
    // 64 rows 52 to 49 us, 80 rows 74 to 64 (16 requests: 21.5 to 23.6, 28.4 to 29.5); width 128: 32 rows 56 to 67, 48 rows 103 to 70; width 256: 16 rows 100 to
    // 170, 24 rows 184 to 171.
    p.tile = rows > (W == 64 ? 64 : W == 128 ? 32 : 16);
    p.min_units = 4;
    if (!p.tile) {
        // 32 rows in one pass or 16 in each of two (64 requests of 2048: 20 rows of width 64 28 to 44 us); for up to 16 rows the smaller tile (25.8 to 27.8)
        p.nr = rows > 16 ? 2 : 1;
        p.max_tiles = (int32_t)up(rows, 16 * p.nr);
        // two resident workgroups per compute unit (64 requests of 4096, width 128: 86.4 us; one 89, three 104, four 97; width 64: 45.6, 49.1, 52.3, 49.3);
        // at least four units for each, a round of its waves (one request of 8192: 13.1 us; one unit 13.7, eight 14.4)
        int64_t grid = 2 * kCus;
        // short caches: four waves are through a row's units in a few rounds, which is less than a second launch takes (one request of 1024 tokens, whole against
        // cut: width 64 8.5 to 10.5 us, 128 11.5 to 12.3, 256 18.2 to 15.0; of 512: 14.2 to 14.9 there; of 2048: 12.1 to 10.6, 17 to 12.6)
        p.whole = max_units <= (W <= 128 ? 16 : 8);
        if (p.whole) p.min_units = 1;
        const int64_t most = p.whole ? B * heads_kv * p.max_tiles : up(B * heads_kv * p.max_tiles * max_units, p.min_units);
        if (grid > most) grid = most;
        p.grid = (int32_t)grid;
        p.splits = 1;
        p.ws_o = 0;
        const int64_t slots = p.whole ? 0 : 2 * grid;
        p.ws_ml = slots * 16 * p.nr * W * 4;
        p.ws_prefix = p.ws_ml + slots * 16 * p.nr * 8;
    } else {
        // 128 rows per workgroup, or 64 where no request has more: 64 requests of 2048 tokens, width 128: 64 rows 72 us (with 128: 87), 80 rows 129 (88); width 256:
        // 178 (267), 330 (269); four prompts of 2048 over 8192, width 256, f16: 536 TFLOP/s with 64, 576 with 128 (590
        // since its weights carry the value scale)
        p.nr = rows > 64 ? 2 : 1;
        const int64_t rows_wg = 64 * p.nr, bound = T * group / rows_wg + B;
        int64_t tiles = up(T * group, rows_wg);
        if (tiles < B) tiles = B;                 // (a request with tokens has a tile of its own)
        // Too few workgroups for the chip: the key range is cut until each compute unit has as many as it holds (two, one above width 128), down to parts of two
        // units, or of sixteen where every compute unit has a workgroup already.  Width 128, 1 / 2 / 4 / 8 / 16 / 32 parts: 64 tokens of group 4 over 16384: 428 225
        // 120 69 47 44 us; 512 over 8192: 215 125 94 105 129 182; twice 512 over 8192: 222 166 171; 8 times 128 over 1024: 37 44 55; 256 over 512: 22 21 20 24.
        const int64_t wgs = tiles * heads_kv, parts = up(max_units, wgs < kCus ? 2 : 16);
        int64_t splits = (W <= 128 ? 2 : 1) * kCus / wgs;
        if (splits > 32) splits = 32;
        if (splits > parts) splits = parts;
        if (splits < 1) splits = 1;
        if (bound * heads_kv * splits > kMaxGrid) return fail(FA_ERR_TOO_LARGE, "more than 2^23 row tiles");
        p.max_tiles = (int32_t)bound;
        p.splits = (int32_t)splits;
        p.grid = (int32_t)(bound * heads_kv * splits);
        const int64_t slots = splits > 1 ? bound * heads_kv * splits : 0;
        p.ws_ml = slots * rows_wg * W * 4;
        p.ws_prefix = p.ws_ml + slots * rows_wg * 8;
    }
    const bool joined = p.tile ? p.splits > 1 : !p.whole;
    if (!p.tile && joined && B * heads_kv > kMaxGrid) return fail(FA_ERR_TOO_LARGE, "more than 2^23 requests times key/value heads");
    // (the join wants a workgroup per compute unit: eight tokens over 16384, width 128: 28.8 us with a quarter of that, 23.6; eight times as many 24.3)
    const int64_t tile_rows = (p.tile ? 64 : 16) * p.nr, most_rows = rows < tile_rows ? rows : tile_rows, items = heads_kv * (p.tile ? p.max_tiles : B * p.max_tiles) * (W / 64);
    p.join_rows = 16;
    while (p.join_rows > 1 && items * up(most_rows, p.join_rows) < kCus) p.join_rows /= 2;
    p.join_chunks = (int32_t)up(most_rows, p.join_rows);
    p.bytes = joined ? p.ws_prefix + 8 * (B + 1) : 0;         // (nothing is parked without a join)
    *out = p;
    return FA_OK;
}

}  // namespace

extern "C" {

int fa_qk_norm_rope_fwd(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight, const void* k_weight, int32_t weight_dtype,
                        const float* table, int64_t table_rows, const void* positions, int32_t position_bytes, int64_t position_stride, int64_t B, int64_t L,
                        int64_t heads, int64_t heads_kv, int64_t D, int64_t R, const int64_t strides[4][3], int32_t dtype, float eps, int32_t interleaved,
                        void* stream) {
    if (!q || !k || !q_out || !k_out || !strides) return fail(FA_ERR_NULL_POINTER, "fa_qk_norm_rope_fwd: null pointer");
    RopeCall c;
    if (int rc = rope_common(&c, q_weight, k_weight, weight_dtype, table, table_rows, positions, position_bytes, position_stride, B, L, heads, heads_kv, D, R, strides, 4,
                             dtype, eps, interleaved))
        return rc;
    const void* in[2] = {q, k};
    void* out[2] = {q_out, k_out};
    for (int i = 0; i < 2; ++i) {
        fa::RopeSide& s = c.p.side[i];
        s.x = in[i]; s.y = out[i];
        s.x_sb = strides[i][0]; s.x_sh = strides[i][1]; s.x_sl = strides[i][2];
        s.y_sb = strides[2 + i][0]; s.y_sh = strides[2 + i][1]; s.y_sl = strides[2 + i][2];
        if (!aligned(in[i], 16) || !aligned(out[i], 16)) c.vec = false;
        if (!aligned(in[i], c.es) || !aligned(out[i], c.es)) return fail(FA_ERR_MISALIGNED, "operands must be aligned to their element size");
    }
    rope_shape(&c, B, false);
    return launched(fa::launch_rope_fwd(c.p, dtype, c.vec, c.hc, c.stream_past, (hipStream_t)stream));
}

int64_t fa_qk_norm_rope_workspace(int64_t B, int64_t L, int64_t heads, int64_t heads_kv, int64_t D) {
    (void)heads; (void)heads_kv;
    if (B < 1 || L < 1 || D < 2) return 0;
    return 2ll * kRopeMaxBlocks * D * 4;
}

int fa_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq, void* dk, const void* q_weight, const void* k_weight,
                        void* dq_weight, void* dk_weight, int32_t weight_dtype, void* workspace, int64_t workspace_bytes, const float* table, int64_t table_rows,
                        const void* positions, int32_t position_bytes, int64_t position_stride, int64_t B, int64_t L, int64_t heads, int64_t heads_kv,
                        int64_t D, int64_t R, const int64_t strides[6][3], int32_t dtype, float eps, int32_t interleaved, void* stream) {
    if (!q || !k || !dq_out || !dk_out || !dq || !dk || !strides) return fail(FA_ERR_NULL_POINTER, "fa_qk_norm_rope_bwd: null pointer");
    if ((dq_weight || dk_weight) && !workspace) return fail(FA_ERR_NULL_POINTER, "fa_qk_norm_rope_bwd: weight gradients need a workspace");
    RopeCall c;
    if (int rc = rope_common(&c, q_weight ? q_weight : dq_weight, k_weight ? k_weight : dk_weight, weight_dtype, table, table_rows, positions, position_bytes,
                             position_stride, B, L, heads, heads_kv, D, R, strides, 6, dtype, eps, interleaved))
        return rc;
    if ((dq_weight || dk_weight) && (workspace_bytes < fa_qk_norm_rope_workspace(B, L, heads, heads_kv, D) || !aligned(workspace, 8)))
        return fail(FA_ERR_WORKSPACE, "fa_qk_norm_rope_bwd: workspace must be 8-byte aligned and hold %lld bytes", (long long)fa_qk_norm_rope_workspace(B, L, heads, heads_kv, D));
    const void* in[2] = {q, k};
    const void* din[2] = {dq_out, dk_out};
    void* out[2] = {dq, dk};
    const void* w[2] = {q_weight, k_weight};
    void* dw[2] = {dq_weight, dk_weight};
    for (int i = 0; i < 2; ++i) {
        fa::RopeSide& s = c.p.side[i];
        s.x = in[i]; s.dy = din[i]; s.y = out[i]; s.w = w[i]; s.dw = dw[i];
        s.dw_part = dw[i] ? (float*)workspace + (int64_t)i * kRopeMaxBlocks * D : nullptr;
        s.x_sb = strides[i][0]; s.x_sh = strides[i][1]; s.x_sl = strides[i][2];
        s.dy_sb = strides[2 + i][0]; s.dy_sh = strides[2 + i][1]; s.dy_sl = strides[2 + i][2];
        s.y_sb = strides[4 + i][0]; s.y_sh = strides[4 + i][1]; s.y_sl = strides[4 + i][2];
        if (!aligned(in[i], 16) || !aligned(din[i], 16) || !aligned(out[i], 16)) c.vec = false;
        if (!aligned(in[i], c.es) || !aligned(din[i], c.es) || !aligned(out[i], c.es)) return fail(FA_ERR_MISALIGNED, "operands must be aligned to their element size");
    }
    rope_shape(&c, B, true);
    return launched(fa::launch_rope_bwd(c.p, dtype, c.vec, c.hc, c.stream_past, (hipStream_t)stream));
}

int fa_cache_tables(const int32_t* seq_lens, const int32_t* new_lens, int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int32_t* free_blocks,
                    int64_t pool_size, const int32_t* free_count, int64_t num_requests, int64_t num_tokens, int64_t block_size, int32_t* seq_lens_out,
                    int32_t* free_count_out, int32_t* cu_new, int32_t* granted, int32_t* positions, int32_t* slots, void* stream) {
    if (!seq_lens || !new_lens || !block_tables || !free_blocks || !free_count || !seq_lens_out || !free_count_out || !cu_new || !granted)
        return fail(FA_ERR_NULL_POINTER, "fa_cache_tables: null pointer");
    if (num_tokens > 0 && (!positions || !slots)) return fail(FA_ERR_NULL_POINTER, "fa_cache_tables: null pointer");
    const int shift = block_shift(block_size);
    if (shift < 0) return fail(FA_ERR_BAD_SHAPE, "block size must be 16, 32, 64 or 128 (got %lld)", (long long)block_size);
    if (num_requests < 1 || num_tokens < 0 || max_blocks < 1 || pool_size < 1) return fail(FA_ERR_BAD_SHAPE, "requests, table width and pool must be >= 1, tokens >= 0");
    if (num_requests > (1 << 24) || num_tokens > kMaxCount || pool_size > kMaxCount || max_blocks > kMaxCount) return fail(FA_ERR_TOO_LARGE, "more than 2^24 requests or 2^30 tokens or blocks");
    if (pool_size * block_size > 0x7fffffffll || max_blocks * block_size > 0x7fffffffll) return fail(FA_ERR_TOO_LARGE, "more than 2^31 - 1 slots");
    if (table_stride < max_blocks || table_stride >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "table stride must hold a row");
    fa::TablesParams p{};
    p.seq_in = seq_lens; p.new_lens = new_lens; p.tables = block_tables; p.pool = free_blocks; p.free_in = free_count; p.free_out = free_count_out;
    p.seq_out = seq_lens_out; p.cu_new = cu_new; p.granted = granted; p.positions = positions; p.slots = slots; p.table_stride = table_stride;
    p.B = (int32_t)num_requests; p.width = (int32_t)max_blocks; p.T = (int32_t)num_tokens; p.shift = shift; p.pool_size = (int32_t)pool_size;
    // one launch while a workgroup places the tokens in a few rounds of 1024 (64 requests: 1024 tokens 6.9 us, with a second launch 9.2; 4096: 9.1 to 9.3; 8192: 11.9 to
    // 9.5; one request: 4.4 to 6.2, 5.2 to 6.3, 6.4 to 6.5)
    p.fused = num_tokens <= 4096;
    return launched(fa::launch_cache_tables(p, (hipStream_t)stream));
}

int fa_cache_append(const void* k, const void* v, const int32_t* slots, void* k_cache, void* v_cache, float* k_scale, float* v_scale, int64_t num_tokens,
                    int64_t heads_kv, int64_t D, int64_t W, int64_t num_blocks, int64_t block_size, const int64_t token_strides[4], const int64_t block_strides[4],
                    int32_t dtype, void* stream) {
    if (!k || !v || !slots || !k_cache || !v_cache || !k_scale || !v_scale || !token_strides || !block_strides) return fail(FA_ERR_NULL_POINTER, "fa_cache_append: null pointer");
    if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return fail(FA_ERR_BAD_DTYPE, "keys and values must be FA_DTYPE_F16 or FA_DTYPE_BF16 (got %d)", dtype);
    if (int rc = cache_geometry(num_blocks, heads_kv, block_size, D, W, block_strides, k_cache, v_cache)) return rc;
    if (num_tokens < 0) return fail(FA_ERR_BAD_SHAPE, "num_tokens must be >= 0");
    if (num_tokens > kMaxCount || num_tokens * heads_kv > 32 * kMaxGrid) return fail(FA_ERR_TOO_LARGE, "more than 2^28 rows of keys");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(FA_ERR_MISALIGNED, "keys and values must be 16-byte aligned");
    for (int i = 0; i < 4; ++i) {
        if (token_strides[i] < 0 || token_strides[i] >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "stride %lld is negative or too large", (long long)token_strides[i]);
        if (token_strides[i] % 8) return fail(FA_ERR_MISALIGNED, "rows of keys and values must be 16-byte aligned");
    }
    if (num_tokens == 0) return FA_OK;
    fa::AppendParams p{};
    p.x[0] = k; p.x[1] = v; p.cache[0] = k_cache; p.cache[1] = v_cache; p.scale[0] = k_scale; p.scale[1] = v_scale; p.slots = slots;
    for (int i = 0; i < 2; ++i) {
        p.x_st[i] = token_strides[2 * i]; p.x_sh[i] = token_strides[2 * i + 1];
        p.block_stride[i] = block_strides[i]; p.scale_stride[i] = block_strides[2 + i];
    }
    p.T = (int32_t)num_tokens; p.H = (int32_t)heads_kv; p.D = (int32_t)D; p.W = (int32_t)W; p.shift = block_shift(block_size);
    p.limit = num_blocks * block_size;
    // tokens per workgroup: about 1024 workgroups in all, which the chip holds at once.  Steps of single tokens spread over the chip (64 tokens of 8 heads of 128: 5.4 us
    // with 4, 12 with 16, 40 with 64), prompts do not pay for workgroups in which no run begins (16384 tokens: 82 us with 4, 51 with 16, 22 with 64;
    // 2048: 13.6, 8.8 and 8.0, with 32 6.2).
    int window = 4;
    while (window < 64 && up(num_tokens, window) * 2 * heads_kv > 1024) window *= 2;
    p.window = window;
    return launched(fa::launch_cache_append(p, dtype, (hipStream_t)stream));
}

int64_t fa_cache_attn_workspace(int64_t num_requests, int64_t num_tokens, int64_t heads, int64_t heads_kv, int64_t D, int64_t block_size, int64_t max_blocks,
                                int64_t max_q_len) {
    fa::CacheAttnPlan plan;
    if (int rc = attn_plan(num_requests, num_tokens, heads, heads_kv, D, block_size, max_blocks, max_q_len, &plan)) return rc;
    return plan.bytes;
}

int fa_cache_attn(const void* q, void* out, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, const int32_t* block_tables,
                  const int32_t* seq_lens, const int32_t* cu_q, void* workspace, int64_t workspace_bytes, int64_t num_requests, int64_t num_tokens, int64_t heads,
                  int64_t heads_kv, int64_t D, int64_t W, int64_t num_blocks, int64_t block_size, int64_t max_blocks, int64_t table_stride, int64_t max_q_len,
                  const int64_t token_strides[4], const int64_t block_strides[4], int32_t dtype, float softmax_scale, void* stream) {
    return fa_cache_attn_granted(q, out, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, nullptr, workspace, workspace_bytes, num_requests, num_tokens, heads,
                                 heads_kv, D, W, num_blocks, block_size, max_blocks, table_stride, max_q_len, token_strides, block_strides, dtype, softmax_scale, stream);
}

int fa_cache_attn_granted(const void* q, void* out, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, const int32_t* block_tables,
                          const int32_t* seq_lens, const int32_t* cu_q, const int32_t* granted, void* workspace, int64_t workspace_bytes, int64_t num_requests, int64_t num_tokens, int64_t heads,
                          int64_t heads_kv, int64_t D, int64_t W, int64_t num_blocks, int64_t block_size, int64_t max_blocks, int64_t table_stride, int64_t max_q_len,
                          const int64_t token_strides[4], const int64_t block_strides[4], int32_t dtype, float softmax_scale, void* stream) {
    if (!q || !out || !k_cache || !v_cache || !k_scale || !v_scale || !block_tables || !seq_lens || !cu_q || !token_strides || !block_strides)
        return fail(FA_ERR_NULL_POINTER, "fa_cache_attn: null pointer");
    if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return fail(FA_ERR_BAD_DTYPE, "queries must be FA_DTYPE_F16 or FA_DTYPE_BF16 (got %d)", dtype);
    fa::CacheAttnPlan plan;
    if (int rc = attn_plan(num_requests, num_tokens, heads, heads_kv, D, block_size, max_blocks, max_q_len, &plan)) return rc;
    if (int rc = cache_geometry(num_blocks, heads_kv, block_size, D, W, block_strides, k_cache, v_cache)) return rc;
    const float scale_log2 = softmax_scale * 1.44269504088896340736f;
    if (!(softmax_scale > 0.f) || !isfinite(scale_log2)) return fail(FA_ERR_BAD_SCALE, "softmax_scale must be > 0 and finite in powers of two (got %g)", (double)softmax_scale);
    if (table_stride < max_blocks || table_stride >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "table stride must hold a row");
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(FA_ERR_MISALIGNED, "queries and output must be 16-byte aligned");
    for (int i = 0; i < 4; ++i) {
        if (token_strides[i] < 0 || token_strides[i] >= kMaxStride) return fail(FA_ERR_BAD_STRIDE, "stride %lld is negative or too large", (long long)token_strides[i]);
        if (token_strides[i] % 8) return fail(FA_ERR_MISALIGNED, "rows of queries and output must be 16-byte aligned");
    }
    if (num_tokens == 0) return FA_OK;
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || !aligned(workspace, 16)))
        return fail(FA_ERR_WORKSPACE, "fa_cache_attn: workspace must be 16-byte aligned and hold %lld bytes", (long long)plan.bytes);
    fa::CacheAttnParams p{};
    p.q = q; p.o = out; p.k = (const uint8_t*)k_cache; p.v = (const uint8_t*)v_cache; p.ks = k_scale; p.vs = v_scale;
    p.tables = block_tables; p.seq_lens = seq_lens; p.cu_q = cu_q; p.granted = granted;
    if (plan.bytes) {
        p.ws_o = (float*)((char*)workspace + plan.ws_o);
        p.ws_ml = (float*)((char*)workspace + plan.ws_ml);
        p.ws_prefix = (long long*)((char*)workspace + plan.ws_prefix);
    }
    p.q_st = token_strides[0]; p.q_sh = token_strides[1]; p.o_st = token_strides[2]; p.o_sh = token_strides[3];
    p.k_bs = block_strides[0]; p.v_bs = block_strides[1]; p.ks_bs = block_strides[2]; p.vs_bs = block_strides[3]; p.table_stride = table_stride;
    p.num_blocks = (int32_t)num_blocks; p.B = (int32_t)num_requests; p.T = (int32_t)num_tokens; p.Hq = (int32_t)heads; p.Hkv = (int32_t)heads_kv;
    p.group = (int32_t)(heads / heads_kv); p.D = (int32_t)D; p.width = (int32_t)max_blocks; p.shift = block_shift(block_size);
    p.grid = plan.grid; p.min_units = plan.min_units; p.whole = plan.whole; p.splits = plan.splits; p.max_tiles = plan.max_tiles; p.join_rows = plan.join_rows; p.join_chunks = plan.join_chunks;
    p.scale_log2 = scale_log2;
    return launched(fa::launch_cache_attn(p, plan, dtype, (hipStream_t)stream));
}

}  // extern "C"
