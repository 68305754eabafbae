// Argument blocks and launchers of the operators around attention over an 8-bit key/value cache (fa_rope.hip, fa_cache_update.hip,
// fa_cache_attn.hip) and their C entry points (fa_cache_capi.cpp).
//
// Cache layout.  A block holds P tokens (16, 32, 64 or 128) of every key/value head; W = head dim rounded up to a multiple of 64.
//   k_cache [blocks][heads][P][W]   one e4m3 byte per value: a token's row is contiguous, as the key operand of Q K^T wants it
//   v_cache [blocks][heads][W][P]   token-inner: a lane of the P V product finds sixteen tokens of one column in one 16-byte load, so the
//                                   attention kernels need no transpose between memory and the matrix pipe
//   k_scale, v_scale [blocks][heads] float32; value = code * scale
// Blocks are addressed through their own 64-bit stride, everything inside a block through 32-bit offsets.
#ifndef FA_CACHE_H
#define FA_CACHE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {

// ---- norm of every query / key head with the position rotation (fa_rope.hip); index 0 = queries, 1 = keys -----------------------------
struct RopeSide {
    const void* x;          // input rows
    const void* dy;         // backward: gradient of the output rows
    void* y;                // forward: output rows; backward: gradient of the input rows
    const void* w;          // [D] or null (ones)
    void* dw;               // backward: [D] or null
    float* dw_part;         // backward: [blocks][D] partial sums
    int64_t x_sb, x_sh, x_sl, dy_sb, dy_sh, dy_sl, y_sb, y_sh, y_sl;   // strides in elements: batch, head, row
    int32_t heads;
    int32_t chunks;         // head chunks per token: ceil(heads / heads per lane group)
    int32_t items;          // tokens * chunks
    int32_t blocks;         // workgroups
    int32_t head_inner;     // consecutive lane groups take: 1 = the chunks of one token, 0 = the tokens of one chunk
};
struct RopeParams {
    RopeSide side[2];
    const float* table;     // [table_rows][R]: R / 2 cosines, then R / 2 sines
    const void* positions;  // int32 or int64, or null: the row's index
    int64_t table_rows, pos_sb;   // pos_sb: elements between two batch entries' positions (0 = shared)
    int32_t pos64, L, D, R, interleaved, w_f32;
    float eps;
};
// vec: 16-byte accesses; stream_past: the data does not fit the last cache and is not kept there
hipError_t launch_rope_fwd(const RopeParams& p, int dtype, bool vec, int heads_per_group, bool stream_past, hipStream_t stream);
hipError_t launch_rope_bwd(const RopeParams& p, int dtype, bool vec, int heads_per_group, bool stream_past, hipStream_t stream);

// ---- block tables, positions and slots of one step (fa_cache_update.hip) --------------------------------------------------------------
struct TablesParams {
    const int32_t* seq_in;  // [B] tokens held (may be seq_out)
    const int32_t* new_lens;// [B] tokens that come; negative = the request ends
    int32_t* tables;        // [B][width] (row stride table_stride)
    int32_t* pool;          // [pool_size] free blocks: pool[0 .. free_in - 1]
    const int32_t* free_in;
    int32_t* free_out;      // may be free_in
    int32_t* seq_out;       // [B]
    int32_t* cu_new;        // [B + 1]
    int32_t* granted;       // [B]
    int32_t* positions;     // [T]
    int32_t* slots;         // [T]
    int64_t table_stride;
    int32_t B, width, T, shift, pool_size;
    int32_t fused;          // 1: the one workgroup of the first kernel writes positions and slots too
};
hipError_t launch_cache_tables(const TablesParams& p, hipStream_t stream);

// ---- new keys and values into the cache (fa_cache_update.hip) -------------------------------------------------------------------------
struct AppendParams {
    const void* x[2];       // [T][H][D] keys, values
    void* cache[2];
    float* scale[2];
    const int32_t* slots;   // [T]; negative = padding
    int64_t x_st[2], x_sh[2];        // token, head strides in elements
    int64_t block_stride[2];         // bytes between two blocks
    int64_t scale_stride[2];         // elements between two blocks' scales
    int64_t limit;          // number of slots: blocks * P
    int32_t T, H, D, W, shift, window;
};
hipError_t launch_cache_append(const AppendParams& p, int dtype, hipStream_t stream);

// ---- attention over the cache (fa_cache_attn.hip) -------------------------------------------------------------------------------------
struct CacheAttnParams {
    const void* q;          // [T][Hq][D]
    void* o;                // [T][Hq][D]
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* tables;  // [B][width]
    const int32_t* seq_lens;// [B]
    const int32_t* cu_q;    // [B + 1]
    const int32_t* granted; // [B] or null; 0 = the request's rows see nothing
    float* ws_o;            // partial sums, see fa_cache_attn.hip
    float* ws_ml;
    long long* ws_prefix;   // [B + 1]
    int64_t q_st, q_sh, o_st, o_sh;
    int64_t k_bs, v_bs, ks_bs, vs_bs, table_stride;
    int32_t num_blocks, B, T, Hq, Hkv, group, D, width, shift;
    int32_t grid;           // workgroups of the row kernel
    int32_t min_units;      // fewest 64-token units that are worth a workgroup
    int32_t whole;          // row kernel: no row tile is cut, none is joined
    int32_t splits;         // tile kernel: parts of a tile's key range
    int32_t max_tiles;      // tile kernel: bound on the row tiles of one key/value head
    int32_t join_rows, join_chunks;   // join kernel: rows of a workgroup (1 .. 16), workgroups that share the rows of a tile
    float scale_log2;
};
struct CacheAttnPlan {
    int32_t tile;           // 0 = row kernel (few query rows per key/value head), 1 = tile kernel
    int32_t nr;             // 16-row query tiles per wave
    int32_t width;          // W
    int32_t grid, splits, max_tiles, min_units, whole, join_rows, join_chunks;
    int64_t ws_o, ws_ml, ws_prefix, bytes;   // workspace offsets in bytes and its size
};
hipError_t launch_cache_attn(const CacheAttnParams& p, const CacheAttnPlan& plan, int dtype, hipStream_t stream);

// text of the last failure on this thread (fa_capi.cpp); returns `code`
int set_error(int code, const char* text);

}  // namespace fa
#endif
