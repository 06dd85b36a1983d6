// kvb_api_kv8.cuh -- launchers and C entry points of the 8-bit KV cache and of the
// shared-prefix decode attention (part of kvb_api.cu's translation unit, which holds
// the library's device code).
#pragma once

namespace kvb {

static bool valid_kv_format(int f) { return f == KVB_KV_INT8 || f == KVB_KV_E4M3; }

// Calls F<T, kFmt>(args...) for the run-time dtype and cache format.
#define KVB_KV8_DISPATCH(F, dtype, fmt, ...)                                   \
    ((dtype) == KVB_BF16                                                       \
         ? ((fmt) == KVB_KV_INT8 ? F<__nv_bfloat16, KVB_KV_INT8>(__VA_ARGS__)  \
                                 : F<__nv_bfloat16, KVB_KV_E4M3>(__VA_ARGS__)) \
         : ((fmt) == KVB_KV_INT8 ? F<__half, KVB_KV_INT8>(__VA_ARGS__)         \
                                 : F<__half, KVB_KV_E4M3>(__VA_ARGS__)))

// ---------------------------------------------------------------- argument checks
// Contiguous cache: sequence b's rows at b * seq_stride / head_dim, [n_kv][max_seq].
static int kv8_place_contiguous(const char* name, Kv8Place& c, const void* kc, const void* vc,
                                const float* ks, const float* vs, size_t seq_stride,
                                size_t cache_len, size_t scale_len, size_t n_seq, size_t n_kv,
                                size_t head_dim, size_t max_seq) {
    KVB_CHECK(head_dim > 0 && head_dim <= 256 && n_kv > 0,
              "%s: head_dim %zu must be in 1..256 and n_kv > 0", name, head_dim);
    KVB_CHECK(fits_i32(n_seq) && fits_i32(n_kv) && fits_i32(max_seq) && fits_i32(n_kv * max_seq),
              "%s: a dimension does not fit in i32", name);
    const size_t per_seq = n_kv * max_seq * head_dim;
    KVB_CHECK(seq_stride >= per_seq && seq_stride % head_dim == 0,
              "%s: seq_stride %zu must be a multiple of head_dim and at least %zu", name,
              seq_stride, per_seq);
    KVB_CHECK(n_seq == 0 ||
                  (cache_len >= per_seq && (n_seq == 1 || (cache_len - per_seq) / (n_seq - 1) >= seq_stride)),
              "%s: cache of %zu elems is too small", name, cache_len);
    KVB_CHECK(cache_len % head_dim == 0 && scale_len == cache_len / head_dim,
              "%s: %zu scales for a cache of %zu elems, want one per %zu", name, scale_len,
              cache_len, head_dim);
    KVB_CHECK(kc != nullptr && vc != nullptr && ks != nullptr && vs != nullptr,
              "%s: null cache or scales", name);
    memset(&c, 0, sizeof c);
    c.kc = static_cast<uint8_t*>(const_cast<void*>(kc));
    c.vc = static_cast<uint8_t*>(const_cast<void*>(vc));
    c.ks = const_cast<float*>(ks);
    c.vs = const_cast<float*>(vs);
    c.seq_rows = (long long)(seq_stride / head_dim);
    c.n_kv = (int)n_kv;
    c.hd = (int)head_dim;
    c.max_seq = (int)max_seq;
    return KVB_OK;
}

static int kv8_place_paged(const char* name, Kv8Place& c, const void* k_pool, const void* v_pool,
                           const float* k_scales, const float* v_scales, size_t pool_len,
                           size_t scale_len, const int32_t* block_table, size_t max_blocks,
                           size_t block_size, size_t n_seq, size_t n_kv, size_t head_dim) {
    KVB_CHECK(head_dim > 0 && head_dim <= 256 && n_kv > 0,
              "%s: head_dim %zu must be in 1..256 and n_kv > 0", name, head_dim);
    KVB_CHECK(block_table != nullptr, "%s: null block table", name);
    KVB_CHECK(block_size > 0 && fits_i32(block_size) && fits_i32(n_kv) &&
                  fits_i32(n_kv * block_size) && fits_i32(max_blocks) &&
                  fits_i32(max_blocks * block_size) && fits_i32(n_seq) &&
                  fits_i32(n_seq * max_blocks),
              "%s: a dimension does not fit in i32 (or block_size is 0)", name);
    const size_t per_block = n_kv * block_size * head_dim;
    KVB_CHECK(pool_len % per_block == 0 && fits_i32(pool_len / per_block),
              "%s: pool of %zu elems is not a whole number of %zu-elem blocks", name, pool_len,
              per_block);
    KVB_CHECK(scale_len == pool_len / head_dim,
              "%s: %zu scales for a pool of %zu elems, want one per %zu", name, scale_len, pool_len,
              head_dim);
    KVB_CHECK(k_pool != nullptr && v_pool != nullptr && k_scales != nullptr && v_scales != nullptr,
              "%s: null pool or scales", name);
    memset(&c, 0, sizeof c);
    c.kc = static_cast<uint8_t*>(const_cast<void*>(k_pool));
    c.vc = static_cast<uint8_t*>(const_cast<void*>(v_pool));
    c.ks = const_cast<float*>(k_scales);
    c.vs = const_cast<float*>(v_scales);
    c.n_kv = (int)n_kv;
    c.hd = (int)head_dim;
    c.max_seq = (int)(max_blocks * block_size);
    c.block_table = block_table;
    c.max_blocks = (int)max_blocks;
    c.block_size = (int)block_size;
    c.n_blocks = (int)(pool_len / per_block);
    return KVB_OK;
}

// ---------------------------------------------------------------- append
template <typename T, int kFmt>
static int launch_kv8_append(kvb_stream_t stream, const Kv8AppendArgs& a, size_t rows) {
    if ((a.c.hd == 64 || a.c.hd == 128) && aligned(a.qkv, 16) && aligned(a.cos_t, 16) &&
        aligned(a.sin_t, 16) && aligned(a.c.kc, 8) && aligned(a.c.vc, 8)) {
        const int cpr = a.c.hd / 16;
        const long long items = (long long)(a.n_q + 2 * a.c.n_kv) * cpr;
        const unsigned threads = items >= 256 ? 256u : (unsigned)((items + 31) / 32 * 32);
        const cudaError_t e =
            cpr == 4 ? launch_pdl(kv8_append_vec_kernel<T, kFmt, 4>, dim3((unsigned)rows),
                                  dim3(threads), 0, stream, a)
                     : launch_pdl(kv8_append_vec_kernel<T, kFmt, 8>, dim3((unsigned)rows),
                                  dim3(threads), 0, stream, a);
        return e == cudaSuccess ? KVB_OK : cuda_fail(e, "rope_kv_append_q8 launch");
    }
    const long long items = (long long)rows * (a.n_q + 2 * a.c.n_kv);
    const long long grid = (items + 3) / 4;
    KVB_CHECK(grid <= 0x7fffffffll, "rope_kv_append_q8: too many rows");
    kv8_append_general_kernel<T, kFmt><<<(unsigned)grid, 128, 0, stream>>>(a, items);
    KVB_CHECK_LAUNCH("rope_kv_append_q8 launch");
    return KVB_OK;
}

static int kv8_append(const char* name, kvb_stream_t stream, void* qkv, size_t qkv_len,
                      size_t n_seq, size_t t, const int32_t* pos, const float* cos_t,
                      const float* sin_t, size_t table_len, const Kv8Place& c, size_t n_q,
                      int kv_format, int dtype) {
    const size_t hd = (size_t)c.hd, stride = (n_q + 2 * (size_t)c.n_kv) * hd;
    KVB_CHECK(hd % 2 == 0, "%s: odd head_dim %zu", name, hd);
    KVB_CHECK(fits_i32(n_q) && fits_i32(stride) && fits_i32(t) && fits_i32(n_seq * t),
              "%s: a dimension does not fit in i32", name);
    KVB_CHECK(qkv_len == n_seq * t * stride, "%s: qkv has %zu elems, want %zux%zux%zu", name,
              qkv_len, n_seq, t, stride);
    KVB_CHECK((cos_t == nullptr) == (sin_t == nullptr), "%s: one of cos / sin is null", name);
    KVB_CHECK(!cos_t || (table_len % (hd / 2) == 0 && fits_i32(table_len / (hd / 2))),
              "%s: bad cos/sin table sizes", name);
    if (n_seq == 0 || t == 0) return KVB_OK;
    KVB_CHECK(qkv != nullptr && pos != nullptr, "%s: null qkv or position array", name);
    Kv8AppendArgs a;
    a.qkv = static_cast<uint16_t*>(qkv);
    a.n_q = (int)n_q;
    a.row_stride = (int)stride;
    a.rows_per_seq = (int)t;
    a.pos = pos;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.max_pos = cos_t ? (int)(table_len / (hd / 2)) : 0;
    a.c = c;
    return KVB_KV8_DISPATCH(launch_kv8_append, dtype, kv_format, stream, a, n_seq * t);
}

// ---------------------------------------------------------------- read back
template <typename T, int kFmt>
static int launch_kv8_read(kvb_stream_t stream, const Kv8ReadArgs& a, size_t n_seq) {
    const int chunks = a.c.hd / 16;
    const long long per_head = (long long)a.t * chunks;
    if (a.c.hd % 16 == 0 && n_seq * a.c.n_kv <= 65535 && per_head <= 0x7fffff00ll &&
        aligned(a.c.kc, 16) && aligned(a.c.vc, 16) && aligned(a.k_out, 16) && aligned(a.v_out, 16)) {
        const dim3 grid((unsigned)((per_head + 255) / 256), (unsigned)(n_seq * a.c.n_kv));
        const cudaError_t e =
            launch_pdl(kv8_read_vec_kernel<T, kFmt>, grid, dim3(256), 0, stream, a, chunks);
        return e == cudaSuccess ? KVB_OK : cuda_fail(e, "kv_read_q8 launch");
    }
    const long long items = (long long)n_seq * a.t * a.c.n_kv * 2;
    const long long grid = (items + 3) / 4;
    KVB_CHECK(grid <= 0x7fffffffll, "kv_read_q8: too many rows");
    kv8_read_general_kernel<T, kFmt><<<(unsigned)grid, 128, 0, stream>>>(a, items);
    KVB_CHECK_LAUNCH("kv_read_q8 launch");
    return KVB_OK;
}

static int kv8_read(const char* name, kvb_stream_t stream, const Kv8Place& c, const int32_t* pos,
                    size_t n_seq, size_t t, void* k_out, void* v_out, size_t out_len,
                    size_t out_rows, int kv_format, int dtype) {
    KVB_CHECK(fits_i32(t) && fits_i32(out_rows) && fits_i32(n_seq * t),
              "%s: a dimension does not fit in i32", name);
    KVB_CHECK(t <= out_rows, "%s: %zu rows into outputs of %zu", name, t, out_rows);
    KVB_CHECK(out_len == n_seq * (size_t)c.n_kv * out_rows * (size_t)c.hd,
              "%s: outputs of %zu elems, want %zux%dx%zux%d", name, out_len, n_seq, c.n_kv,
              out_rows, c.hd);
    if (n_seq == 0 || t == 0) return KVB_OK;
    KVB_CHECK(pos != nullptr && k_out != nullptr && v_out != nullptr,
              "%s: null positions or outputs", name);
    Kv8ReadArgs a;
    a.c = c;
    a.pos = pos;
    a.t = (int)t;
    a.out_rows = (int)out_rows;
    a.k_out = static_cast<uint16_t*>(k_out);
    a.v_out = static_cast<uint16_t*>(v_out);
    return KVB_KV8_DISPATCH(launch_kv8_read, dtype, kv_format, stream, a, n_seq);
}

// ---------------------------------------------------------------- decode attention
static int decode_args(const char* name, GeneralDecodeArgs& a, const void* q, size_t q_row_stride,
                       const int32_t* lens, size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                       size_t head_dim, float scale, void* out, size_t out_row_stride) {
    KVB_CHECK(n_kv > 0 && n_q > 0 && n_q % n_kv == 0, "%s: n_q %zu not a multiple of n_kv %zu", name,
              n_q, n_kv);
    KVB_CHECK(head_dim > 0 && head_dim <= 256, "%s: head_dim %zu must be in 1..256", name, head_dim);
    KVB_CHECK(fits_i32(n_seq) && fits_i32(max_len) && fits_i32(n_q * head_dim),
              "%s: a dimension does not fit in i32", name);
    KVB_CHECK(q_row_stride >= n_q * head_dim, "%s: q_row_stride too small", name);
    KVB_CHECK(out_row_stride >= n_q * head_dim, "%s: out_row_stride too small", name);
    KVB_CHECK(n_seq == 0 || (q != nullptr && lens != nullptr && out != nullptr),
              "%s: null q, lengths or output", name);
    a.q = static_cast<const uint16_t*>(q);
    a.q_row_stride = (long long)q_row_stride;
    a.lens = lens;
    a.max_len = (int)max_len;
    a.n_q = (int)n_q;
    a.n_kv = (int)n_kv;
    a.hd = (int)head_dim;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.out = static_cast<uint16_t*>(out);
    a.out_row_stride = (long long)out_row_stride;
    return KVB_OK;
}

// 2-D tensor map of `rows` rows of row_bytes 8-bit elements, copied box_rows at a time;
// swizzled over the row (64 or 128 bytes).
static int encode_tmap_rows8(CUtensorMap* map, const void* base, size_t row_bytes, size_t rows,
                             int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(KVB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {row_bytes, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)row_bytes, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims,
                          strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(KVB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return KVB_OK;
}

static bool q8_tensor_shape(size_t head_dim, size_t n_q, size_t n_kv) {
    return (head_dim == 64 || head_dim == 128) && n_kv > 0 && n_q % n_kv == 0 &&
           n_q / n_kv <= (size_t)kQ8MaxGroup;
}

// Keys per CTA of a split call.  The fewest tiles, up to 20, with which one wave of three CTAs
// per SM holds the worst case (every sequence at max_len); beyond that about five waves, of
// at least 20 tiles: shorter chunks pay more starts and a longer join, longer ones leave a
// longer last wave.  Pairs of (sequence, KV head) that fill the SMs by themselves with at most
// 32 tiles take one chunk each and no join; so do 12 tiles (768 keys of 64 dims) in any case:
// one sequence of 513 keys 5.7 us in a graph against 5.3 in three chunks, but 9.6 against 12.2
// where the host launches it, as the second launch is 2 us of the host's time.  Against the best of 4 to 128 tiles over 140 shapes
// (full and ragged batches, n_kv 1 to 8, both head_dims) 3.9 % slower on average, 24 % at worst.
// Measured on B200, tiles per CTA: one sequence x 8 heads at 65536 keys 12 / 16 / 20 / 32:
// 23.5 / 25.0 / 19.5 / 22.2 us (16 is a wave and a bit); 16 x 8 at 4096 8 / 16 / 20 / 32: 22.3 /
// 23.3 / 18.1 / 20.9; 64 x 8 U[1,4096] 8 / 16 / 20 / 48: 37.4 / 33.8 / 35.1 / 34.9; 32 x 8 at 1000
// keys 8 / 12 / 16: 16.4 / 13.7 / 12.3.  At most kJoinMaxParts chunks.
static int q8_chunk_keys(size_t n_seq, size_t n_kv, size_t max_len, size_t head_dim) {
    const size_t kt = (size_t)q8_tile_keys((int)head_dim);
    const size_t tiles = (max_len + kt - 1) / kt, pairs = n_seq * n_kv;
    const size_t slots = (size_t)num_sms() * kQ8CtasPerSm;
    const size_t chunks = pairs < slots && pairs > 0 ? slots / pairs : 1;  // of a pair, in one wave
    size_t per_cta = (tiles + chunks - 1) / chunks;
    if (per_cta > 20) {
        per_cta = (pairs * tiles + 5 * slots - 1) / (5 * slots);
        if (per_cta < 20) per_cta = 20;
    }
    if (tiles <= 12 || (pairs >= (size_t)num_sms() && tiles <= 32)) per_cta = tiles;
    if (per_cta * kJoinMaxParts < tiles) per_cta = (tiles + kJoinMaxParts - 1) / kJoinMaxParts;
    if (per_cta > tiles) per_cta = tiles;
    if (per_cta < 1) per_cta = 1;
    return (int)((per_cta + kQ8Warps - 1) / kQ8Warps * kQ8Warps * kt);
}

static size_t q8_ws_bytes(size_t n_seq, size_t max_len, size_t n_q, size_t n_kv, size_t head_dim) {
    if (!q8_tensor_shape(head_dim, n_q, n_kv) || max_len == 0) return 0;
    const size_t ck = (size_t)q8_chunk_keys(n_seq, n_kv, max_len, head_dim);
    const size_t chunks = (max_len + ck - 1) / ck;
    return chunks <= 1 ? 0
                       : n_seq * n_kv * chunks * q8_part_floats((int)(n_q / n_kv), (int)head_dim) *
                             sizeof(float);
}

// Chunks of a split call, in a workspace and joined by a pass.  (A fold through a cluster, as
// kvb_attention_decode has for small grids, measured slower in 560 of 565 of them, by 13 % on
// average: 8 sequences x 8 heads at 2000 keys 10.0 us, the join 9.0.)
struct Q8Plan {
    int chunk_keys, max_chunks;
};
static Q8Plan q8_plan(size_t n_seq, size_t max_len, size_t n_q, size_t n_kv, size_t head_dim,
                      const void* ws, size_t ws_len) {
    const size_t unit = (size_t)kQ8Warps * q8_tile_keys((int)head_dim);
    const bool split = q8_ws_bytes(n_seq, max_len, n_q, n_kv, head_dim) > 0 && ws != nullptr &&
                       aligned(ws, 16);
    size_t ck = (max_len + unit - 1) / unit * unit;  // one chunk
    if (split) {  // a smaller workspace takes fewer and longer chunks
        const size_t fit = ws_len / (n_seq * n_kv * q8_part_floats((int)(n_q / n_kv), (int)head_dim) *
                                     sizeof(float));
        const size_t want = (size_t)q8_chunk_keys(n_seq, n_kv, max_len, head_dim);
        if (fit >= (max_len + want - 1) / want) ck = want;
        else if (fit >= 2) ck = ((max_len + fit - 1) / fit + unit - 1) / unit * unit;
    }
    if (ck == 0) ck = unit;
    Q8Plan p;
    p.chunk_keys = (int)ck;
    p.max_chunks = max_len ? (int)((max_len + ck - 1) / ck) : 1;
    return p;
}

template <typename T, int HD>
static int launch_join(kvb_stream_t stream, const JoinArgs& a, size_t n_seq) {
    // parts that one load a lane reaches, and the warps of 16 loads that reach all of them
    const int side = 128 / HD;
    const int w = a.max_parts <= 16 * side ? 1 : a.max_parts <= 32 * side ? 2
                  : a.max_parts <= 64 * side ? 4 : 8;
    const int rows = kJoinWarps / w;
    const dim3 grid((unsigned)((a.n_kv * a.group + rows - 1) / rows), (unsigned)n_seq);
    auto* kernel = a.max_parts <= 8 * side ? attn_join_kernel<T, HD, 1, 8>
                   : w == 1                ? attn_join_kernel<T, HD, 1, 16>
                   : w == 2                ? attn_join_kernel<T, HD, 2, 16>
                   : w == 4                ? attn_join_kernel<T, HD, 4, 16>
                                           : attn_join_kernel<T, HD, 8, 16>;
    const cudaError_t e = launch_pdl(kernel, grid, dim3(32 * kJoinWarps), 0, stream, a);
    return e == cudaSuccess ? KVB_OK : cuda_fail(e, "attention join launch");
}

template <typename T, int kFmt, int HD, int NT>
static int launch_q8_tensor(kvb_stream_t stream, Q8DecodeArgs& a, size_t n_seq, size_t cache_rows,
                            void* ws, size_t ws_len) {
    constexpr int KT = q8_tile_keys(HD);
    a.piece = KT;
    if (a.c.block_table)
        while (a.c.block_size % a.piece) a.piece /= 2;
    a.bs_shift = -1;
    for (int s = 0; a.c.block_table && s < 31; ++s)
        if (a.c.block_size == 1 << s) a.bs_shift = s;
    a.total_rows = (int)cache_rows;
    CUtensorMap kmap, vmap;
    int st = encode_tmap_rows8(&kmap, a.c.kc, HD, cache_rows, a.piece);
    if (st) return st;
    st = encode_tmap_rows8(&vmap, a.c.vc, HD, cache_rows, a.piece);
    if (st) return st;
    const size_t n_kv = (size_t)a.c.n_kv;
    const Q8Plan plan = q8_plan(n_seq, (size_t)a.max_len, n_kv * a.group, n_kv, HD, ws, ws_len);
    a.chunk_keys = plan.chunk_keys;
    a.max_chunks = plan.max_chunks;
    a.ws = plan.max_chunks > 1 ? static_cast<float*>(ws) : nullptr;
    auto* kernel = a.rope_cos ? attn_decode_q8_kernel<T, kFmt, HD, NT, true>
                              : attn_decode_q8_kernel<T, kFmt, HD, NT, false>;
    set_max_smem(kernel, kQ8SmemBytes);
    const dim3 grid((unsigned)n_kv, (unsigned)n_seq, (unsigned)a.max_chunks);
    const cudaError_t e =
        launch_pdl(kernel, grid, dim3(kQ8Warps * 32), (size_t)kQ8SmemBytes, stream, kmap, vmap, a);
    if (e != cudaSuccess) return cuda_fail(e, "attention_decode_q8 launch");
    if (a.max_chunks == 1) return KVB_OK;
    JoinArgs j;
    j.ws = a.ws;
    j.lens = a.lens;
    j.max_len = a.max_len;
    j.key0 = 0;
    j.chunk_keys = a.chunk_keys;
    j.fixed = 0;
    j.max_parts = a.max_chunks;
    j.part_floats = q8_part_floats(a.group, HD);
    j.n_kv = a.c.n_kv;
    j.group = a.group;
    j.write_all = 0;
    j.prefix = 0;
    j.out = a.out;
    j.out_row_stride = a.out_row_stride;
    return launch_join<T, HD>(stream, j, n_seq);
}

// The tensor-core kernel where shape and alignment allow it (cache_rows: rows of the code
// arrays), else the general one; with RoPE tables (the fused form) else KVB_ERR_UNSUPPORTED.
struct Q8Rope {
    const float* cos_t = nullptr;
    const float* sin_t = nullptr;
    int max_pos = 0;
    bool kv_ready = false;  // Q8DecodeArgs::kv_ready
};
template <typename T, int kFmt>
static int launch_q8_decode(kvb_stream_t stream, const GeneralDecodeArgs& a, const Kv8Place& c,
                            size_t cache_rows, size_t n_seq, void* ws, size_t ws_len,
                            const Q8Rope& rope) {
    const bool tensor = q8_tensor_shape((size_t)a.hd, (size_t)a.n_q, (size_t)a.n_kv) &&
                        (!c.block_table || c.block_size % 16 == 0) && a.q_row_stride % 4 == 0 &&
                        aligned(a.q, 8) && aligned(c.kc, 16) && aligned(c.vc, 16) &&
                        aligned(c.ks, 4) && aligned(c.vs, 4) && n_seq <= 65535 &&
                        a.n_kv <= 65535 && cache_rows > 0 && fits_i32(cache_rows + 64) &&
                        a.max_len <= 1 << 30;
    if (rope.cos_t && !(tensor && aligned(rope.cos_t, 16) && aligned(rope.sin_t, 16)))
        return fail(KVB_ERR_UNSUPPORTED,
                    "rope_attention_decode_q8: needs head_dim 64 or 128, n_q/n_kv <= 16, block_size "
                    "a multiple of 16 and 16-byte aligned caches and tables (use "
                    "kvb_rope_kv_append_q8 + kvb_attention_decode_q8)");
    if (!tensor) {
        Q8Source<T, kFmt> src;
        src.c = c;
        const dim3 grid((unsigned)n_seq, (unsigned)((a.n_q + 3) / 4));
        attn_general_src_kernel<T, Q8Source<T, kFmt>><<<grid, 128, 0, stream>>>(a, src);
        KVB_CHECK_LAUNCH("attention_decode_q8 launch");
        return KVB_OK;
    }
    Q8DecodeArgs d;
    d.q = a.q;
    d.q_row_stride = a.q_row_stride;
    d.lens = a.lens;
    d.max_len = a.max_len;
    d.group = a.n_q / a.n_kv;
    d.scale_log2 = a.scale_log2;
    d.out = a.out;
    d.out_row_stride = a.out_row_stride;
    d.c = c;
    d.rope_cos = rope.cos_t;
    d.rope_sin = rope.sin_t;
    d.rope_max_pos = rope.max_pos;
    d.kv_ready = rope.kv_ready ? 1 : 0;
    if (a.hd == 64)
        return d.group <= 8 ? launch_q8_tensor<T, kFmt, 64, 1>(stream, d, n_seq, cache_rows, ws, ws_len)
                            : launch_q8_tensor<T, kFmt, 64, 2>(stream, d, n_seq, cache_rows, ws, ws_len);
    return d.group <= 8 ? launch_q8_tensor<T, kFmt, 128, 1>(stream, d, n_seq, cache_rows, ws, ws_len)
                        : launch_q8_tensor<T, kFmt, 128, 2>(stream, d, n_seq, cache_rows, ws, ws_len);
}

// How a shared-prefix call runs on the tensor-core kernels: the prefix's 64-key tiles dealt to
// `splits` slices, the sequences' rows to tiles of which a CTA takes `groups`, the own keys in
// chunks.
struct SharedPlan {
    int key0;  // keys computed for all sequences at once
    int seqs_per_tile, row_tiles, groups, n_tiles, splits;
    int chunk_keys, max_chunks, part_floats;
    size_t ws_bytes;
};
// A workspace for a larger call may be a little small for this one: then fewer slices, and own
// keys in longer chunks; ws_bytes is above ws_len only where not even one of each fits.
static SharedPlan shared_plan(size_t n_seq, size_t prefix, size_t max_own, size_t n_q, size_t n_kv,
                              size_t ws_len) {
    SharedPlan p;
    const size_t group = n_q / n_kv;
    p.key0 = (int)prefix;
    p.seqs_per_tile = (int)(kSpRows / group);
    p.row_tiles = (int)((n_seq + p.seqs_per_tile - 1) / p.seqs_per_tile);
    p.n_tiles = (int)((prefix + kSpKeys - 1) / kSpKeys);
    p.groups = p.row_tiles >= 3 ? 4 : p.row_tiles;
    p.splits = 0;
    // Slices: the number that takes the least time by a model fitted on B200 (us; 28 shapes x 1 to
    // 64 slices, n_kv 1 to 8, both types: the choice is 1.8 % slower than the best on average,
    // 12 % at worst).  A slice takes 0.77 + 0.19 per row tile that shares its SM for each 64-key
    // tile, and 3.6 to start and end.  All slices and the own keys (half of the worst case, at
    // 5.75 TB/s) share the SMs, and a seventh of a slice's time is not covered by the own keys.
    // A slice adds its rows' partials (264 bytes written and read, 3.1 TB/s) to the join.  32
    // sequences, 4096 keys, 128 own, by slices 4 / 8 / 16 / 32: 22.0 / 15.8 / 12.7 / 13.7 us; 256
    // sequences, 16384 keys, up to 1000 own, 4 / 6 / 12 / 24: 124 / 97 / 107 / 133.
    const size_t pairs = (size_t)((p.row_tiles + p.groups - 1) / p.groups) * n_kv;
    const size_t sms = (size_t)num_sms(), most_ctas = (size_t)(kSpMaxGroups / p.groups);
    const double own_us = 0.5 * (double)n_seq * (double)max_own * (double)n_kv * 256.0 / 5.75e6;
    const double join_us = 0.007 + (double)n_seq * (double)n_q * 264.0 * 2.0 / 3.1e6;
    double best = 1e30;
    for (int s = 1; s <= p.n_tiles && s <= 64; ++s) {
        const size_t ctas = pairs * s;
        const size_t per_sm = ctas >= most_ctas * sms ? most_ctas : (ctas + sms - 1) / sms;
        const double slice =
            (0.77 + 0.19 * (double)(p.groups * per_sm)) * ((p.n_tiles + s - 1) / s) + 3.6;
        const double waves = (double)((ctas + per_sm * sms - 1) / (per_sm * sms));
        const double share = (double)ctas * slice / (double)(per_sm * sms) + own_us;
        const double cost =
            (share > waves * slice ? share : waves * slice) + 0.15 * slice + s * join_us;
        if (cost < best) {
            best = cost;
            p.splits = s;
        }
    }
    size_t ck = max_own ? (size_t)decode_chunk_keys(n_seq, n_kv, max_own) : 256;
    p.part_floats = q8_part_floats((int)group, 64);
    const size_t part_bytes = n_seq * n_kv * (size_t)p.part_floats * sizeof(float);
    const size_t fit = part_bytes ? ws_len / part_bytes : 0;  // parts of a (sequence, KV head)
    size_t chunks = (max_own + ck - 1) / ck;
    if ((size_t)p.splits + chunks > fit && p.splits > 1)
        p.splits = fit > chunks + 1 ? (int)(fit - chunks) : 1;
    size_t most = kJoinMaxParts - 64;
    if (fit > (size_t)p.splits && fit - p.splits < most) most = fit - p.splits;
    if (chunks > most) ck = ((max_own + most - 1) / most + 255) / 256 * 256;
    p.chunk_keys = (int)ck;
    p.max_chunks = (int)((max_own + ck - 1) / ck);
    p.ws_bytes = part_bytes * (size_t)(p.splits + p.max_chunks);
    return p;
}

template <typename T, int kGroups>
static int launch_shared_prefix(kvb_stream_t stream, const CUtensorMap& qmap, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, const SharedPrefixArgs& s) {
    auto* kernel = s.lens ? attn_shared_prefix_kernel<T, kGroups, true>
                          : attn_shared_prefix_kernel<T, kGroups, false>;
    set_max_smem(kernel, sp_smem_bytes(kGroups));
    const dim3 grid((unsigned)s.n_kv, (unsigned)s.splits,
                    (unsigned)((s.row_tiles + kGroups - 1) / kGroups));
    const cudaError_t e = launch_pdl(kernel, grid, dim3(sp_threads(kGroups)),
                                     (size_t)sp_smem_bytes(kGroups), stream, qmap, kmap, vmap, s);
    return e == cudaSuccess ? KVB_OK : cuda_fail(e, "attention_decode_shared prefix launch");
}

template <typename T>
static int launch_shared_tensor(kvb_stream_t stream, const GeneralDecodeArgs& a,
                                const SharedSource<T>& src, const SharedPlan& p, size_t n_seq,
                                size_t own_rows, float* ws) {
    const int group = a.n_q / a.n_kv, max_parts = p.splits + p.max_chunks;
    const bool paged = src.block_table != nullptr;
    const int dtype = Elem<T>::kDtype;
    const size_t total_rows =
        paged ? (size_t)src.n_blocks * src.n_kv * src.block_size : own_rows;
    if (p.splits > 0) {
        CUtensorMap qmap, kmap, vmap;
        {
            const uint64_t dims[3] = {64, (uint64_t)a.n_q, n_seq};
            const uint64_t strides[2] = {128, (uint64_t)a.q_row_stride * 2};
            const uint32_t box[3] = {64, (uint32_t)group, (uint32_t)p.seqs_per_tile};
            const int st = encode_tmap(&qmap, a.q, 3, dims, strides, box, dtype);
            if (st) return st;
        }
        int st;
        if (paged) {
            const uint64_t dims[2] = {64, total_rows}, strides[1] = {128};
            const uint32_t box[2] = {64, (uint32_t)kSpKeys};
            st = encode_tmap(&kmap, src.kc, 2, dims, strides, box, dtype);
            if (!st) st = encode_tmap(&vmap, src.vc, 2, dims, strides, box, dtype);
        } else {
            const uint64_t dims[3] = {64, (uint64_t)p.key0, (uint64_t)a.n_kv};
            const uint64_t strides[2] = {128, (uint64_t)src.prefix_rows * 128};
            const uint32_t box[3] = {64, (uint32_t)kSpKeys, 1};
            st = encode_tmap(&kmap, src.pk, 3, dims, strides, box, dtype);
            if (!st) st = encode_tmap(&vmap, src.pv, 3, dims, strides, box, dtype);
        }
        if (st) return st;
        SharedPrefixArgs s;
        s.n_seq = (int)n_seq;
        s.n_kv = a.n_kv;
        s.group = group;
        s.seqs_per_tile = p.seqs_per_tile;
        s.row_tiles = p.row_tiles;
        s.prefix = p.key0;
        s.n_tiles = p.n_tiles;
        s.splits = p.splits;
        s.scale_log2 = a.scale_log2;
        s.lens = paged ? a.lens : nullptr;
        s.max_len = a.max_len;
        s.ws = ws;
        s.max_parts = max_parts;
        s.part_floats = p.part_floats;
        s.block_table = src.block_table;
        s.block_size = src.block_size;
        s.n_blocks = src.n_blocks;
        st = p.groups == 4   ? launch_shared_prefix<T, 4>(stream, qmap, kmap, vmap, s)
             : p.groups == 2 ? launch_shared_prefix<T, 2>(stream, qmap, kmap, vmap, s)
                             : launch_shared_prefix<T, 1>(stream, qmap, kmap, vmap, s);
        if (st) return st;
    }
    if (p.max_chunks > 0) {
        CUtensorMap kmap, vmap;
        const uint64_t dims[2] = {64, total_rows}, strides[1] = {128};
        const uint32_t box[2] = {64, 64};
        int st = encode_tmap(&kmap, src.kc, 2, dims, strides, box, dtype);
        if (!st) st = encode_tmap(&vmap, src.vc, 2, dims, strides, box, dtype);
        if (st) return st;
        DecodeArgs d = {};
        d.q = a.q;
        d.q_row_stride = a.q_row_stride;
        d.lens = a.lens;
        d.max_len = a.max_len;
        d.n_kv = a.n_kv;
        d.group = group;
        d.max_seq = src.max_seq;
        d.seq_rows = src.seq_rows;
        d.scale_log2 = a.scale_log2;
        d.ws = ws;
        d.chunk_keys = p.chunk_keys;
        d.max_chunks = p.max_chunks;
        d.block_table = src.block_table;
        d.max_blocks = src.max_blocks;
        d.block_size = src.block_size;
        d.n_blocks = src.n_blocks;
        d.key0 = paged ? p.key0 : 0;
        d.part0 = p.splits;
        d.max_parts = max_parts;
        d.part_floats = p.part_floats;
        auto* kernel = attn_decode_part_kernel<T>;
        set_max_smem(kernel, kDecSmemBytes);
        const dim3 grid((unsigned)a.n_kv, (unsigned)n_seq, (unsigned)p.max_chunks);
        cudaError_t e;
        if (p.splits > 0) {
            e = launch_pdl(kernel, grid, dim3(128), kDecSmemBytes, stream, kmap, vmap, d);
        } else {  // no kernel before it that has waited for the ones before: an ordinary launch
            kernel<<<grid, 128, kDecSmemBytes, stream>>>(kmap, vmap, d);
            e = cudaGetLastError();
        }
        if (e != cudaSuccess) return cuda_fail(e, "attention_decode_shared launch");
    }
    JoinArgs j;
    j.ws = ws;
    j.lens = a.lens;
    j.max_len = a.max_len;
    j.key0 = paged ? p.key0 : 0;
    j.chunk_keys = p.chunk_keys;
    j.fixed = p.splits;
    j.max_parts = max_parts;
    j.part_floats = p.part_floats;
    j.n_kv = a.n_kv;
    j.group = group;
    j.write_all = 1;
    j.prefix = paged ? 0 : src.prefix;
    j.out = a.out;
    j.out_row_stride = a.out_row_stride;
    return launch_join<T, 64>(stream, j, n_seq);
}

// The most keys that the own kernel of a paged call has of a sequence, `shared` (whole tiles) by the
// prefix's: one at least where a sequence may end inside the prefix.
static size_t shared_paged_own(size_t max_len, size_t shared) {
    return max_len > shared ? max_len - shared : shared > 0 ? 1 : 0;
}

// The tensor-core kernels where shape, alignment and workspace allow them (own_rows: rows of 64
// elements of the contiguous caches), else the general kernel.
template <typename T>
static int launch_shared(kvb_stream_t stream, const GeneralDecodeArgs& a, const SharedSource<T>& src,
                         size_t n_seq, size_t own_rows, void* ws, size_t ws_len) {
    const bool paged = src.block_table != nullptr;
    if (a.hd == 64 && a.n_q / a.n_kv <= kQ8MaxGroup && a.scale_log2 > 0.f &&
        a.q_row_stride % 8 == 0 && aligned(a.q, 16) &&
        aligned(src.kc, 16) && aligned(src.vc, 16) && aligned(src.pk, 16) && aligned(src.pv, 16) &&
        n_seq <= 65535 && a.n_kv <= 65535 && a.max_len <= 1 << 30 && src.prefix <= 1 << 30 &&
        ws != nullptr && aligned(ws, 16) &&
        (paged ? src.block_size % 64 == 0 && src.n_blocks > 0 &&
                     fits_i32((size_t)src.n_blocks * src.n_kv * src.block_size + 64)
               : fits_i32(own_rows + 64))) {
        // Paged: whole 64-key tiles of the prefix for all at once; each sequence reads the rest
        // through its own table row.  Contiguous: all of the prefix.
        const size_t shared = paged ? (size_t)src.prefix / 64 * 64 : (size_t)src.prefix;
        const size_t own = paged ? shared_paged_own(a.max_len, shared) : (size_t)a.max_len;
        const SharedPlan p =
            shared_plan(n_seq, shared, own, (size_t)a.n_q, (size_t)a.n_kv, ws_len);
        // (no keys at all: no kernel of this call for the join to follow)
        if (ws_len >= p.ws_bytes && p.splits + p.max_chunks > 0)
            return launch_shared_tensor<T>(stream, a, src, p, n_seq, own_rows,
                                           static_cast<float*>(ws));
    }
    const dim3 grid((unsigned)n_seq, (unsigned)((a.n_q + 3) / 4));
    attn_general_src_kernel<T, SharedSource<T>><<<grid, 128, 0, stream>>>(a, src);
    KVB_CHECK_LAUNCH("attention_decode_shared launch");
    return KVB_OK;
}

int q8_join_launches(size_t n_seq, size_t max_len, size_t n_q, size_t n_kv, size_t head_dim,
                     const void* ws, size_t ws_len) {
    if (!q8_tensor_shape(head_dim, n_q, n_kv) || n_seq == 0) return 0;
    const Q8Plan p = q8_plan(n_seq, max_len, n_q, n_kv, head_dim, ws, ws_len);
    return p.max_chunks > 1 ? 1 : 0;
}

}  // namespace kvb

extern "C" {

int kvb_rope_kv_append_q8(kvb_stream_t stream, void* qkv, size_t qkv_len, size_t n_seq, size_t t,
                          const int32_t* pos, const float* cos_t, const float* sin_t,
                          size_t table_len, void* kc, void* vc, float* ks, float* vs,
                          size_t seq_stride, size_t cache_len, size_t scale_len, size_t n_q,
                          size_t n_kv, size_t head_dim, size_t max_seq, int kv_format, int dtype) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    Kv8Place c;
    const int st = kv8_place_contiguous("rope_kv_append_q8", c, kc, vc, ks, vs, seq_stride,
                                        cache_len, scale_len, n_seq, n_kv, head_dim, max_seq);
    if (st) return st;
    return kv8_append("rope_kv_append_q8", stream, qkv, qkv_len, n_seq, t, pos, cos_t, sin_t,
                      table_len, c, n_q, kv_format, dtype);
}

int kvb_rope_kv_append_q8_paged(kvb_stream_t stream, void* qkv, size_t qkv_len, size_t n_seq,
                                size_t t, const int32_t* pos, const float* cos_t,
                                const float* sin_t, size_t table_len, void* k_pool, void* v_pool,
                                float* k_scales, float* v_scales, size_t pool_len, size_t scale_len,
                                const int32_t* block_table, size_t max_blocks, size_t block_size,
                                size_t n_q, size_t n_kv, size_t head_dim, int kv_format,
                                int dtype) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    Kv8Place c;
    const int st = kv8_place_paged("rope_kv_append_q8_paged", c, k_pool, v_pool, k_scales, v_scales,
                                   pool_len, scale_len, block_table, max_blocks, block_size, n_seq,
                                   n_kv, head_dim);
    if (st) return st;
    return kv8_append("rope_kv_append_q8_paged", stream, qkv, qkv_len, n_seq, t, pos, cos_t, sin_t,
                      table_len, c, n_q, kv_format, dtype);
}

int kvb_kv_read_q8(kvb_stream_t stream, const void* kc, const void* vc, const float* ks,
                   const float* vs, size_t seq_stride, size_t cache_len, size_t scale_len,
                   const int32_t* pos, size_t n_seq, size_t t, size_t n_kv, size_t head_dim,
                   size_t max_seq, void* k_out, void* v_out, size_t out_len, size_t out_rows,
                   int kv_format, int dtype) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    Kv8Place c;
    const int st = kv8_place_contiguous("kv_read_q8", c, kc, vc, ks, vs, seq_stride, cache_len,
                                        scale_len, n_seq, n_kv, head_dim, max_seq);
    if (st) return st;
    return kv8_read("kv_read_q8", stream, c, pos, n_seq, t, k_out, v_out, out_len, out_rows,
                    kv_format, dtype);
}

int kvb_kv_read_q8_paged(kvb_stream_t stream, const void* k_pool, const void* v_pool,
                         const float* k_scales, const float* v_scales, size_t pool_len,
                         size_t scale_len, const int32_t* block_table, size_t max_blocks,
                         size_t block_size, const int32_t* pos, size_t n_seq, size_t t, size_t n_kv,
                         size_t head_dim, void* k_out, void* v_out, size_t out_len,
                         size_t out_rows, int kv_format, int dtype) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    Kv8Place c;
    const int st = kv8_place_paged("kv_read_q8_paged", c, k_pool, v_pool, k_scales, v_scales,
                                   pool_len, scale_len, block_table, max_blocks, block_size, n_seq,
                                   n_kv, head_dim);
    if (st) return st;
    return kv8_read("kv_read_q8_paged", stream, c, pos, n_seq, t, k_out, v_out, out_len, out_rows,
                    kv_format, dtype);
}

size_t kvb_attention_decode_q8_workspace_bytes(size_t n_seq, size_t max_len, size_t n_q,
                                               size_t n_kv, size_t head_dim) {
    return q8_ws_bytes(n_seq, max_len, n_q, n_kv, head_dim);
}

static int q8_decode_contiguous(const char* name, kvb_stream_t stream, const void* q,
                                size_t q_row_stride, const void* kc, const void* vc, const float* ks,
                                const float* vs, size_t seq_stride, size_t cache_len,
                                size_t scale_len, const int32_t* lens, size_t n_seq, size_t max_len,
                                size_t n_q, size_t n_kv, size_t head_dim, size_t max_seq,
                                float scale, void* out, size_t out_row_stride, void* workspace,
                                size_t workspace_len, int kv_format, int dtype, const Q8Rope& rope) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    GeneralDecodeArgs a;
    int st = decode_args(name, a, q, q_row_stride, lens, n_seq, max_len, n_q, n_kv, head_dim, scale,
                         out, out_row_stride);
    if (st) return st;
    KVB_CHECK(max_len <= max_seq, "%s: max_len %zu exceeds max_seq %zu", name, max_len, max_seq);
    Kv8Place c;
    st = kv8_place_contiguous(name, c, kc, vc, ks, vs, seq_stride, cache_len, scale_len, n_seq, n_kv,
                              head_dim, max_seq);
    if (st) return st;
    if (n_seq == 0) return KVB_OK;
    const size_t cache_rows = scale_len;
    return KVB_KV8_DISPATCH(launch_q8_decode, dtype, kv_format, stream, a, c, cache_rows, n_seq,
                            workspace, workspace_len, rope);
}

static int q8_decode_paged(const char* name, kvb_stream_t stream, const void* q, size_t q_row_stride,
                           const void* k_pool, const void* v_pool, const float* k_scales,
                           const float* v_scales, size_t pool_len, size_t scale_len,
                           const int32_t* block_table, size_t max_blocks, size_t block_size,
                           const int32_t* lens, size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                           size_t head_dim, float scale, void* out, size_t out_row_stride,
                           void* workspace, size_t workspace_len, int kv_format, int dtype,
                           const Q8Rope& rope) {
    KVB_CHECK_DTYPE(dtype);
    KVB_CHECK(valid_kv_format(kv_format), "unknown KV format %d", kv_format);
    GeneralDecodeArgs a;
    int st = decode_args(name, a, q, q_row_stride, lens, n_seq, max_len, n_q, n_kv, head_dim, scale,
                         out, out_row_stride);
    if (st) return st;
    Kv8Place c;
    st = kv8_place_paged(name, c, k_pool, v_pool, k_scales, v_scales, pool_len, scale_len, block_table,
                         max_blocks, block_size, n_seq, n_kv, head_dim);
    if (st) return st;
    KVB_CHECK(max_len <= max_blocks * block_size, "%s: max_len %zu exceeds %zu blocks of %zu", name,
              max_len, max_blocks, block_size);
    if (n_seq == 0) return KVB_OK;
    const size_t cache_rows = scale_len;
    return KVB_KV8_DISPATCH(launch_q8_decode, dtype, kv_format, stream, a, c, cache_rows, n_seq,
                            workspace, workspace_len, rope);
}

// The fused forms' tables and qkv rows.
static int q8_rope(const char* name, Q8Rope& r, const void* qkv, size_t qkv_len, const float* cos_t,
                   const float* sin_t, size_t table_len, size_t n_seq, size_t n_q, size_t n_kv,
                   size_t head_dim) {
    KVB_CHECK(head_dim > 0 && head_dim % 2 == 0 && head_dim <= 256 && table_len % (head_dim / 2) == 0 &&
                  fits_i32(table_len / (head_dim / 2)),
              "%s: bad head_dim or cos/sin table sizes", name);
    KVB_CHECK(cos_t != nullptr && sin_t != nullptr, "%s: null table", name);
    KVB_CHECK(fits_i32(n_seq) && fits_i32(n_q) && fits_i32(n_kv) &&
                  qkv_len == n_seq * (n_q + 2 * n_kv) * head_dim,
              "%s: qkv has %zu elems, want %zux%zu", name, qkv_len, n_seq,
              (n_q + 2 * n_kv) * head_dim);
    r.cos_t = cos_t;
    r.sin_t = sin_t;
    r.max_pos = (int)(table_len / (head_dim / 2));
    return KVB_OK;
}

int kvb_attention_decode_q8(kvb_stream_t stream, const void* q, size_t q_row_stride, const void* kc,
                            const void* vc, const float* ks, const float* vs, size_t seq_stride,
                            size_t cache_len, size_t scale_len, const int32_t* lens, size_t n_seq,
                            size_t max_len, size_t n_q, size_t n_kv, size_t head_dim,
                            size_t max_seq, float scale, void* out, size_t out_row_stride,
                            void* workspace, size_t workspace_len, int kv_format, int dtype) {
    return q8_decode_contiguous("attention_decode_q8", stream, q, q_row_stride, kc, vc, ks, vs,
                                seq_stride, cache_len, scale_len, lens, n_seq, max_len, n_q, n_kv,
                                head_dim, max_seq, scale, out, out_row_stride, workspace,
                                workspace_len, kv_format, dtype, Q8Rope());
}

int kvb_attention_decode_q8_paged(kvb_stream_t stream, const void* q, size_t q_row_stride,
                                  const void* k_pool, const void* v_pool, const float* k_scales,
                                  const float* v_scales, size_t pool_len, size_t scale_len,
                                  const int32_t* block_table, size_t max_blocks, size_t block_size,
                                  const int32_t* lens, size_t n_seq, size_t max_len, size_t n_q,
                                  size_t n_kv, size_t head_dim, float scale, void* out,
                                  size_t out_row_stride, void* workspace, size_t workspace_len,
                                  int kv_format, int dtype) {
    return q8_decode_paged("attention_decode_q8_paged", stream, q, q_row_stride, k_pool, v_pool,
                           k_scales, v_scales, pool_len, scale_len, block_table, max_blocks, block_size,
                           lens, n_seq, max_len, n_q, n_kv, head_dim, scale, out, out_row_stride,
                           workspace, workspace_len, kv_format, dtype, Q8Rope());
}

static int rope_attention_q8(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                             const float* cos_t, const float* sin_t, size_t table_len, void* kc,
                             void* vc, float* ks, float* vs, size_t seq_stride, size_t cache_len,
                             size_t scale_len, const int32_t* lens, size_t n_seq, size_t max_len,
                             size_t n_q, size_t n_kv, size_t head_dim, size_t max_seq, float scale,
                             void* out, size_t out_row_stride, void* workspace,
                             size_t workspace_len, int kv_format, int dtype, bool kv_ready) {
    Q8Rope r;
    const int st = q8_rope("rope_attention_decode_q8", r, qkv, qkv_len, cos_t, sin_t, table_len, n_seq,
                           n_q, n_kv, head_dim);
    if (st) return st;
    r.kv_ready = kv_ready;
    return q8_decode_contiguous("rope_attention_decode_q8", stream, qkv, (n_q + 2 * n_kv) * head_dim,
                                kc, vc, ks, vs, seq_stride, cache_len, scale_len, lens, n_seq, max_len,
                                n_q, n_kv, head_dim, max_seq, scale, out, out_row_stride, workspace,
                                workspace_len, kv_format, dtype, r);
}

static int rope_attention_q8_paged(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                                   const float* cos_t, const float* sin_t, size_t table_len,
                                   void* k_pool, void* v_pool, float* k_scales, float* v_scales,
                                   size_t pool_len, size_t scale_len, const int32_t* block_table,
                                   size_t max_blocks, size_t block_size, const int32_t* lens,
                                   size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                                   size_t head_dim, float scale, void* out, size_t out_row_stride,
                                   void* workspace, size_t workspace_len, int kv_format, int dtype,
                                   bool kv_ready) {
    Q8Rope r;
    const int st = q8_rope("rope_attention_decode_q8_paged", r, qkv, qkv_len, cos_t, sin_t, table_len,
                           n_seq, n_q, n_kv, head_dim);
    if (st) return st;
    r.kv_ready = kv_ready;
    return q8_decode_paged("rope_attention_decode_q8_paged", stream, qkv, (n_q + 2 * n_kv) * head_dim,
                           k_pool, v_pool, k_scales, v_scales, pool_len, scale_len, block_table,
                           max_blocks, block_size, lens, n_seq, max_len, n_q, n_kv, head_dim, scale,
                           out, out_row_stride, workspace, workspace_len, kv_format, dtype, r);
}

int kvb_rope_attention_decode_q8(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                                 const float* cos_t, const float* sin_t, size_t table_len, void* kc,
                                 void* vc, float* ks, float* vs, size_t seq_stride,
                                 size_t cache_len, size_t scale_len, const int32_t* lens,
                                 size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                                 size_t head_dim, size_t max_seq, float scale, void* out,
                                 size_t out_row_stride, void* workspace, size_t workspace_len,
                                 int kv_format, int dtype) {
    return rope_attention_q8(stream, qkv, qkv_len, cos_t, sin_t, table_len, kc, vc, ks, vs,
                             seq_stride, cache_len, scale_len, lens, n_seq, max_len, n_q, n_kv,
                             head_dim, max_seq, scale, out, out_row_stride, workspace,
                             workspace_len, kv_format, dtype, false);
}

int kvb_rope_attention_decode_q8_paged(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                                       const float* cos_t, const float* sin_t, size_t table_len,
                                       void* k_pool, void* v_pool, float* k_scales, float* v_scales,
                                       size_t pool_len, size_t scale_len,
                                       const int32_t* block_table, size_t max_blocks,
                                       size_t block_size, const int32_t* lens, size_t n_seq,
                                       size_t max_len, size_t n_q, size_t n_kv, size_t head_dim,
                                       float scale, void* out, size_t out_row_stride,
                                       void* workspace, size_t workspace_len, int kv_format,
                                       int dtype) {
    return rope_attention_q8_paged(stream, qkv, qkv_len, cos_t, sin_t, table_len, k_pool, v_pool,
                                   k_scales, v_scales, pool_len, scale_len, block_table, max_blocks,
                                   block_size, lens, n_seq, max_len, n_q, n_kv, head_dim, scale,
                                   out, out_row_stride, workspace, workspace_len, kv_format, dtype,
                                   false);
}

size_t kvb_attention_decode_shared_workspace_bytes(size_t n_seq, size_t shared_len, size_t max_own,
                                                   size_t n_q, size_t n_kv, size_t head_dim) {
    if (head_dim != 64 || n_seq == 0 || n_kv == 0 || n_q % n_kv != 0 || n_q / n_kv == 0 ||
        n_q / n_kv > (size_t)kQ8MaxGroup || !fits_i32(shared_len) || !fits_i32(max_own))
        return 0;
    // contiguous, or paged with the prefix cut to whole 64-key tiles: the larger need
    const size_t a = shared_plan(n_seq, shared_len, max_own, n_q, n_kv, SIZE_MAX).ws_bytes;
    const size_t tiles = shared_len / 64 * 64;
    const size_t b = shared_plan(n_seq, tiles, kvb::shared_paged_own(shared_len + max_own, tiles), n_q,
                                 n_kv, SIZE_MAX).ws_bytes;
    return a > b ? a : b;
}

int kvb_attention_decode_shared(kvb_stream_t stream, const void* q, size_t q_row_stride,
                                const void* pk, const void* pv, size_t prefix_len,
                                size_t prefix_rows, const void* kc, const void* vc,
                                size_t seq_stride, size_t cache_len, const int32_t* lens,
                                size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                                size_t head_dim, size_t max_seq, float scale, void* out,
                                size_t out_row_stride, void* workspace, size_t workspace_len,
                                int dtype) {
    KVB_CHECK_DTYPE(dtype);
    GeneralDecodeArgs a;
    const int st = decode_args("attention_decode_shared", a, q, q_row_stride, lens, n_seq, max_len,
                               n_q, n_kv, head_dim, scale, out, out_row_stride);
    if (st) return st;
    KVB_CHECK(prefix_len <= prefix_rows && fits_i32(n_kv * prefix_rows) &&
                  fits_i32(prefix_len + max_len),
              "attention_decode_shared: prefix of %zu keys in buffers of %zu", prefix_len,
              prefix_rows);
    KVB_CHECK(max_len <= max_seq && fits_i32(max_seq) && fits_i32(n_kv * max_seq),
              "attention_decode_shared: max_len %zu exceeds max_seq %zu", max_len, max_seq);
    const size_t per_seq = n_kv * max_seq * head_dim;
    KVB_CHECK(seq_stride >= per_seq && seq_stride % head_dim == 0,
              "attention_decode_shared: seq_stride %zu must be a multiple of head_dim and at least "
              "%zu", seq_stride, per_seq);
    KVB_CHECK(n_seq == 0 ||
                  (cache_len >= per_seq && (n_seq == 1 || (cache_len - per_seq) / (n_seq - 1) >= seq_stride)),
              "attention_decode_shared: cache of %zu elems is too small", cache_len);
    KVB_CHECK((max_len == 0 || (kc != nullptr && vc != nullptr)) &&
                  (prefix_len == 0 || (pk != nullptr && pv != nullptr)),
              "attention_decode_shared: null cache");
    if (n_seq == 0) return KVB_OK;
    auto go = [&](auto tag) {
        SharedSource<decltype(tag)> s;
        memset(&s, 0, sizeof s);
        s.pk = static_cast<const uint16_t*>(pk);
        s.pv = static_cast<const uint16_t*>(pv);
        s.prefix = (int)prefix_len;
        s.prefix_rows = (int)prefix_rows;
        s.kc = static_cast<const uint16_t*>(kc);
        s.vc = static_cast<const uint16_t*>(vc);
        s.seq_rows = (long long)(seq_stride / head_dim);
        s.n_kv = (int)n_kv;
        s.hd = (int)head_dim;
        s.max_seq = (int)max_seq;
        return launch_shared(stream, a, s, n_seq, cache_len / head_dim, workspace, workspace_len);
    };
    return dtype == KVB_BF16 ? go(__nv_bfloat16()) : go(__half());
}

int kvb_attention_decode_shared_paged(kvb_stream_t stream, const void* q, size_t q_row_stride,
                                      const void* k_pool, const void* v_pool, size_t pool_len,
                                      const int32_t* block_table, size_t max_blocks,
                                      size_t block_size, size_t shared_len, const int32_t* lens,
                                      size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                                      size_t head_dim, float scale, void* out,
                                      size_t out_row_stride, void* workspace, size_t workspace_len,
                                      int dtype) {
    KVB_CHECK_DTYPE(dtype);
    GeneralDecodeArgs a;
    const int st = decode_args("attention_decode_shared_paged", a, q, q_row_stride, lens, n_seq,
                               max_len, n_q, n_kv, head_dim, scale, out, out_row_stride);
    if (st) return st;
    KVB_CHECK(block_table != nullptr, "attention_decode_shared_paged: null block table");
    KVB_CHECK(block_size > 0 && fits_i32(block_size) && fits_i32(n_kv * block_size) &&
                  fits_i32(max_blocks) && fits_i32(max_blocks * block_size) &&
                  fits_i32(n_seq * max_blocks),
              "attention_decode_shared_paged: a dimension does not fit in i32 (or block_size is 0)");
    const size_t per_block = n_kv * block_size * head_dim;
    KVB_CHECK(pool_len % per_block == 0 && fits_i32(pool_len / per_block),
              "attention_decode_shared_paged: pool of %zu elems is not a whole number of %zu-elem "
              "blocks", pool_len, per_block);
    KVB_CHECK(max_len <= max_blocks * block_size && shared_len <= max_blocks * block_size,
              "attention_decode_shared_paged: max_len %zu or shared_len %zu exceeds %zu blocks of %zu",
              max_len, shared_len, max_blocks, block_size);
    KVB_CHECK(k_pool != nullptr && v_pool != nullptr, "attention_decode_shared_paged: null pool");
    if (n_seq == 0) return KVB_OK;
    auto go = [&](auto tag) {
        SharedSource<decltype(tag)> s;
        memset(&s, 0, sizeof s);
        s.prefix = (int)shared_len;
        s.kc = static_cast<const uint16_t*>(k_pool);
        s.vc = static_cast<const uint16_t*>(v_pool);
        s.n_kv = (int)n_kv;
        s.hd = (int)head_dim;
        s.max_seq = (int)(max_blocks * block_size);
        s.block_table = block_table;
        s.max_blocks = (int)max_blocks;
        s.block_size = (int)block_size;
        s.n_blocks = (int)(pool_len / per_block);
        return launch_shared(stream, a, s, n_seq, 0, workspace, workspace_len);
    };
    return dtype == KVB_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // extern "C"

// ------------------------------------------------------------------ decode-step forms
namespace kvb {

int rope_attention_decode_q8_in_step(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                                     const float* cos_t, const float* sin_t, size_t table_len,
                                     void* kc, void* vc, float* ks, float* vs, size_t seq_stride,
                                     size_t cache_len, size_t scale_len, const int32_t* lens,
                                     size_t n_seq, size_t max_len, size_t n_q, size_t n_kv,
                                     size_t head_dim, size_t max_seq, float scale, void* out,
                                     size_t out_row_stride, void* workspace, size_t workspace_len,
                                     int kv_format, int dtype) {
    return ::rope_attention_q8(stream, qkv, qkv_len, cos_t, sin_t, table_len, kc, vc, ks, vs,
                               seq_stride, cache_len, scale_len, lens, n_seq, max_len, n_q, n_kv,
                               head_dim, max_seq, scale, out, out_row_stride, workspace,
                               workspace_len, kv_format, dtype, true);
}

int rope_attention_decode_q8_paged_in_step(kvb_stream_t stream, const void* qkv, size_t qkv_len,
                                           const float* cos_t, const float* sin_t, size_t table_len,
                                           void* k_pool, void* v_pool, float* k_scales,
                                           float* v_scales, size_t pool_len, size_t scale_len,
                                           const int32_t* block_table, size_t max_blocks,
                                           size_t block_size, const int32_t* lens, size_t n_seq,
                                           size_t max_len, size_t n_q, size_t n_kv, size_t head_dim,
                                           float scale, void* out, size_t out_row_stride,
                                           void* workspace, size_t workspace_len, int kv_format,
                                           int dtype) {
    return ::rope_attention_q8_paged(stream, qkv, qkv_len, cos_t, sin_t, table_len, k_pool, v_pool,
                                     k_scales, v_scales, pool_len, scale_len, block_table,
                                     max_blocks, block_size, lens, n_seq, max_len, n_q, n_kv,
                                     head_dim, scale, out, out_row_stride, workspace, workspace_len,
                                     kv_format, dtype, true);
}

}  // namespace kvb
