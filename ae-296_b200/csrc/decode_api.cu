// extern "C" entry points declared in include/b200_decode.h: argument checks and launches only.
#include <cfloat>

#include "decode_common.cuh"

using namespace b200lora;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool rows16(int64_t row, int64_t head) { return row % 8 == 0 && head % 8 == 0; }
bool io_type(int32_t dtype) { return dtype == B200_LORA_F16 || dtype == B200_LORA_BF16; }

int check_cache(const b200_kv_cache* c) {
    if (!c || !c->k || !c->v) return B200_LORA_ERR_NULL;
    if (c->n_pages < 1 || c->page_size < 1 || c->n_kv_heads < 1 || c->head_dim < 1) return B200_LORA_ERR_DIM;
    return B200_LORA_OK;
}

// sizes that do not depend on the launch; 0 or a status
int attention_sizes(AttnParams& p) {
    if (p.a.n_requests < 1 || p.a.n_requests > B200_DECODE_MAX_REQUESTS || p.a.n_groups < 0 || p.a.n_groups > B200_DECODE_MAX_GROUPS ||
        p.a.n_heads < 1 || p.c.n_kv_heads < 1 || p.a.n_heads > 1024 || p.a.n_heads % p.c.n_kv_heads != 0 ||
        (p.c.head_dim != 64 && p.c.head_dim != 128))
        return B200_LORA_ERR_DIM;
    p.per = p.a.n_heads / p.c.n_kv_heads;
    p.per_inverse = (unsigned)(((1ull << 32) + p.per - 1) / p.per);
    p.req_tiles = (p.per + kAttnRows - 1) / kAttnRows;
    p.req_rows = p.per < kAttnRows ? p.per : kAttnRows;
    const int rows = p.a.n_requests * p.per;                  // at most 4096 * 1024
    const bool wide = p.a.n_groups > 0 && rows > kWideFrom;
    // groups of at most kWideFrom rows, and wide ones (of which there are fewer than rows / kWideFrom)
    p.max_group_tiles = p.a.n_groups * (kWideFrom / kAttnRows);
    const int wide_groups = rows / (kWideFrom + 1);
    p.wide_tiles = wide ? (rows + kWideRows - 1) / kWideRows + (p.a.n_groups < wide_groups ? p.a.n_groups : wide_groups) : 0;
    return B200_LORA_OK;
}

size_t attention_bytes(const AttnParams& p) {
    return (attn_group_rows(p) + attn_request_rows(p) + attn_wide_rows(p)) * ((size_t)p.c.head_dim * 4 + 8) +
           4 * ((size_t)4 * p.a.n_groups + p.a.n_requests + 4) + 64;
}

}  // namespace

extern "C" int b200_kv_append(const b200_append* a, const b200_kv_cache* cache, int32_t dtype, void* stream) {
    if (int rc = check_cache(cache)) return rc;
    if (!a || !a->q_out || !a->q || !a->k || !a->v || !a->positions || !a->slots || !a->cos || !a->sin) return B200_LORA_ERR_NULL;
    if (!io_type(dtype)) return B200_LORA_ERR_DTYPE;
    const int d = cache->head_dim, rot = a->rotary_dim;
    if (a->n_tokens < 0 || a->n_heads < 1 || a->n_positions < 1 || d % 2 != 0 || d > 512 || rot < 2 || rot > d || rot % 2 != 0)
        return B200_LORA_ERR_DIM;
    if (a->n_tokens == 0) return B200_LORA_OK;
    // 16-byte vectors where every piece of a unit starts on such a boundary, single elements else
    bool vec = d % 16 == 0 && rot % 16 == 0 && aligned16(a->q_out) && aligned16(a->q) && aligned16(a->k) && aligned16(a->v) &&
               aligned16(cache->k) && aligned16(cache->v) && aligned16(a->cos) && aligned16(a->sin) &&
               rows16(a->q_out_row, a->q_out_head) && rows16(a->q_row, a->q_head) && rows16(a->k_row, a->k_head) && rows16(a->v_row, a->v_head) &&
               rows16(cache->page_stride, cache->token_stride) && cache->head_stride % 8 == 0 &&
               a->table_row % (a->tables_are_f32 ? 4 : 8) == 0;
    if (a->dq) vec = vec && aligned16(a->dq) && rows16(a->dq_row, a->dq_head);
    if (a->dk) vec = vec && aligned16(a->dk) && rows16(a->dk_row, a->dk_head);
    if (a->dv) vec = vec && aligned16(a->dv) && rows16(a->dv_row, a->dv_head);
    const cudaError_t e = launch_kv_append(*a, *cache, dtype, vec, sm_count(), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? B200_LORA_OK : cuda_fail(e);
}

extern "C" size_t b200_prefix_attention_workspace_bytes(int32_t n_requests, int32_t n_groups, int32_t n_heads, int32_t n_kv_heads,
                                                        int32_t head_dim) {
    AttnParams p = {};
    p.a.n_requests = n_requests; p.a.n_groups = n_groups; p.a.n_heads = n_heads;
    p.c.n_kv_heads = n_kv_heads; p.c.head_dim = head_dim;
    return attention_sizes(p) == B200_LORA_OK ? attention_bytes(p) : 0;
}

extern "C" int b200_prefix_attention(const b200_attention* a, const b200_kv_cache* cache, int32_t dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    if (int rc = check_cache(cache)) return rc;
    if (!a || !a->out || !a->q || !a->lens || !workspace) return B200_LORA_ERR_NULL;
    if (a->max_pages > 0 && !a->table) return B200_LORA_ERR_NULL;
    if (a->n_groups > 0 && (!a->prefix_lens || !a->group_starts || (a->max_prefix_pages > 0 && !a->prefix_table))) return B200_LORA_ERR_NULL;
    if (!io_type(dtype)) return B200_LORA_ERR_DTYPE;
    AttnParams p = {};
    p.a = *a; p.c = *cache;
    if (a->n_requests == 0) return B200_LORA_OK;
    if (int rc = attention_sizes(p)) return rc;
    const int ps = cache->page_size;
    if (ps > 256 || (ps & (ps - 1)) != 0 || a->max_pages < 0 || a->max_prefix_pages < 0) return B200_LORA_ERR_DIM;
    // keys of a row of a page table, and units of a cache head in all, are 32-bit numbers
    if ((int64_t)a->max_pages * ps > 0x7fffff00 || (int64_t)a->max_prefix_pages * ps > 0x7fffff00) return B200_LORA_ERR_DIM;
    const int64_t steps = ((int64_t)a->max_pages * ps + kAttnKeys - 1) / kAttnKeys, psteps = ((int64_t)a->max_prefix_pages * ps + kAttnKeys - 1) / kAttnKeys;
    if (steps * p.req_tiles * a->n_requests + psteps * p.max_group_tiles > 0x7fffffff ||
        (psteps / (kWideKeys / kAttnKeys) + 1) * p.wide_tiles > 0x7fffffff)
        return B200_LORA_ERR_DIM;
    if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(cache->k) || !aligned16(cache->v) || !aligned16(workspace) ||
        !rows16(a->q_row, a->q_head) || !rows16(a->out_row, a->out_head) || !rows16(cache->page_stride, cache->token_stride) ||
        cache->head_stride % 8 != 0)
        return B200_LORA_ERR_ALIGN;
    if (workspace_bytes < attention_bytes(p)) return B200_LORA_ERR_WORKSPACE;
    while ((1 << p.page_shift) < ps) ++p.page_shift;
    p.scale_log2 = a->scale * 1.44269504088896341f;
    if (p.scale_log2 == 0.f) p.scale_log2 = FLT_MIN;           // equal weights as before, but what is masked stays at -infinity
    const size_t rows = attn_group_rows(p) + attn_request_rows(p) + attn_wide_rows(p);
    p.part = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part + rows * cache->head_dim);
    p.units = reinterpret_cast<int*>(p.part_ml + rows);
    p.tiles = p.units + a->n_groups + a->n_requests + 1;
    p.wide_units = p.tiles + a->n_groups + 1;
    p.wide_tile = p.wide_units + a->n_groups + 1;
    const cudaError_t e = launch_attention(p, dtype, sm_count(), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? B200_LORA_OK : cuda_fail(e);
}

extern "C" int b200_int4_linear(const b200_int4* a, int32_t dtype, int32_t y_dtype, void* stream) {
    if (!a || !a->y || !a->x || !a->codes || !a->scales) return B200_LORA_ERR_NULL;
    if (!io_type(dtype) || (y_dtype != dtype && y_dtype != B200_LORA_F32)) return B200_LORA_ERR_DTYPE;
    if (a->n_tokens < 0 || a->n_in < 1 || a->n_out < 1 || (a->group != 32 && a->group != 64 && a->group != 128) || a->n_in % a->group != 0)
        return B200_LORA_ERR_DIM;
    if (a->n_in > 0x7fffff00 || a->n_out > 0x7fffff00) return B200_LORA_ERR_DIM;       // rounded up to whole tiles they are 32-bit numbers
    if (!aligned16(a->x) || !aligned16(a->codes) || (a->n_tokens > 1 && a->x_row % 8 != 0)) return B200_LORA_ERR_ALIGN;
    if (a->n_tokens == 0) return B200_LORA_OK;
    b200_int4 q = *a;
    if (a->n_tokens == 1) q.x_row = (a->n_in + 7) / 8 * 8;       // whatever it was said to be
    if (q.x_row < a->n_in || a->n_tokens > 65535 * 32) return B200_LORA_ERR_DIM;      // blocks along z
    const cudaError_t e = launch_int4(q, dtype, y_dtype == B200_LORA_F32, sm_count(), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? B200_LORA_OK : cuda_fail(e);
}
