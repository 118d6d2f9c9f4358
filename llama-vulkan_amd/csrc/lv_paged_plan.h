// lv_paged_plan.h — a paged cache's layout, what its entry points refuse, and how an attention call is dealt to workgroups.  Plain arithmetic,
// for the kernels, the host and tests on machines without a GPU.
#pragma once

#include <stdint.h>

#include "../../include/llava_hip.h"

#if defined(__HIP__) || defined(__HIPCC__)
#define LV_HD __host__ __device__ __forceinline__
#else
#define LV_HD inline
#endif

namespace lv {

// ---- layout ----------------------------------------------------------------------------------------------------------------
constexpr uint32_t kNoPage = 0xffffffffu;

struct PagedView {
    uint8_t *data;
    uint32_t type, kv_heads, dim, shift, pages;   // a page is 1 << shift tokens
    uint32_t code_row, scale_row;                 // bytes of a head's row
    uint32_t half, block;                         // bytes of a block's keys, and of all of it
};

LV_HD PagedView paged_view(const lv_paged_cache &c)
{
    PagedView v{};
    v.data = static_cast<uint8_t *>(c.data);
    v.type = c.type;
    v.kv_heads = c.kv_heads;
    v.dim = c.dim;
    while ((1u << v.shift) < c.page) v.shift++;
    v.pages = c.pages;
    const bool blocks = c.type == LV_Q8_0 || c.type == LV_Q4_0;
    v.code_row = c.type == LV_Q8_0 ? c.dim : c.type == LV_Q4_0 ? c.dim / 2 : 2 * c.dim;
    v.scale_row = blocks ? c.dim / 16 : 0;
    v.half = c.page * (v.code_row + v.scale_row);
    v.block = 2 * v.half;
    return v;
}
// bytes from the pool's start
LV_HD uint64_t paged_codes(const PagedView &v, uint32_t page, uint32_t head, uint32_t which, uint32_t at)
{
    return ((uint64_t)page * v.kv_heads + head) * v.block + (uint64_t)which * v.half + (uint64_t)at * v.code_row;
}
LV_HD uint64_t paged_scales(const PagedView &v, uint32_t page, uint32_t head, uint32_t which, uint32_t at)
{
    return ((uint64_t)page * v.kv_heads + head) * v.block + (uint64_t)which * v.half + ((uint64_t)v.code_row << v.shift) + (uint64_t)at * v.scale_row;
}
// the page of a position, kNoPage where there is none
LV_HD uint32_t paged_page(const PagedView &v, const uint32_t *row, uint32_t table_ld, uint32_t position)
{
    const uint32_t i = position >> v.shift;
    if (i >= table_ld) return kNoPage;
    const uint32_t p = row[i];
    return p < v.pages ? p : kNoPage;
}

// ---- the rows of a sequence ---------------------------------------------------------------------------------------------------
struct PagedSeq {
    uint32_t row0, rows;      // its new tokens' rows
    int32_t pos0;             // position of the first of them; negative where the sequence is shorter than that
    uint32_t keys;            // positions that can be seen: 0 .. keys - 1
};
LV_HD PagedSeq paged_seq(uint32_t start, uint32_t end, uint32_t len, uint32_t tokens, uint32_t positions /* the table's */)
{
    PagedSeq s;
    const uint32_t stop = end < tokens ? end : tokens;
    s.row0 = start;
    s.rows = stop > start ? stop - start : 0;
    // positions are below 2^30; what lies further has no page
    const uint32_t n = len < 0x40000000u ? len : 0x40000000u, m = end > start ? end - start : 0;
    s.pos0 = (int32_t)n - (int32_t)(m < 0x40000000u ? m : 0x40000000u);
    s.keys = n < positions ? n : positions;
    return s;
}

// ---- which keys a position sees -------------------------------------------------------------------------------------------------
LV_HD uint32_t paged_first_key(uint32_t position, uint32_t window, uint32_t chunk)
{
    uint32_t lo = window && position >= window ? position - window + 1 : 0;
    if (chunk) {
        const uint32_t c = position - position % chunk;
        lo = c > lo ? c : lo;
    }
    return lo;
}

// ---- how attention is dealt to workgroups --------------------------------------------------------------------------------------------
// A workgroup takes the queries of one key head in tiles of `tile` rows, a row being a token and one of the `group` heads that share the key head, token
// by token, and some of the keys that they see.  Keys are counted in steps of kPagedStep; a tile that walks `run` steps or up to half as many more is one item, a longer one
// is cut into equal parts of about so many, whose results a second launch puts together.  The run follows from all lengths at once: the steps of all tiles shared
// evenly by as many workgroups as the device holds (`target`), so that one long sequence among short ones is cut finely and equal ones are not cut at all
// when there are enough of them.  A workgroup takes `run_min` steps at least.
// us, 2 or 4 or 8 workgroups a compute unit: 131072 keys of one sequence 99, 106, 111; drafts of 16 sequences 20.4, 21.3, 21.4.
constexpr uint32_t kPagedStep = 128;

struct PagedDeal {
    uint32_t seqs, tokens, group, tile, tile_log2, kv_heads, window, chunk, positions;
    uint32_t target;     // workgroups to share the work; 0: nothing is cut
    uint32_t run_min;    // steps that a workgroup takes at least
};
// steps that a tile of a sequence walks at most: its keys, or as many as a window or a chunk and the tile's tokens cover, and a border on either side
LV_HD uint32_t paged_steps(const PagedDeal &d, const PagedSeq &s)
{
    uint32_t keys = s.keys;
    const uint32_t tokens = d.tile / d.group + 2;
    if (d.window && d.window < keys && d.window + tokens < keys) keys = d.window + tokens;
    if (d.chunk && d.chunk < keys && d.chunk + tokens < keys) keys = d.chunk + tokens;
    return keys == 0 ? 1 : (keys + kPagedStep - 1) / kPagedStep + 1;
}
// `tile` is a power of two; a call's rows, tokens times heads, are fewer than 2^31
LV_HD uint32_t paged_tiles(const PagedDeal &d, const PagedSeq &s) { return (s.rows * d.group + d.tile - 1) >> d.tile_log2; }
// all_steps is a sum of floats, off by less than 1e-4 of itself for 65535 sequences: what that adds to an item count is below the 1 of paged_items
LV_HD uint32_t paged_run(const PagedDeal &d, float all_steps)
{
    if (!d.target) return 0x7fffffffu;
    const float run = all_steps * (float)d.kv_heads / (float)d.target;
    return run < (float)d.run_min ? d.run_min : run > 1e9f ? 1000000000u : (uint32_t)run + 1;
}
LV_HD uint32_t paged_parts(uint32_t steps, uint32_t run)
{
    const uint32_t parts = run > 0x3fffffffu ? 1 : (2 * steps + run) / (2 * run);
    return parts ? parts : 1;
}
// the first of a tile's `steps` that is part p's; its last one's end is p + 1's first
LV_HD uint32_t paged_cut(uint32_t steps, uint32_t p, uint32_t parts) { return (uint32_t)((uint64_t)steps * p / parts); }
// items of a key head at most: parts are no more than steps / run + 1 / 2 a tile, or 1
LV_HD uint64_t paged_items(const PagedDeal &d)
{
    return (uint64_t)d.target / d.kv_heads + 1 + (uint64_t)d.tokens * d.group / d.tile + (d.seqs < d.tokens ? d.seqs : d.tokens);
}

// ---- refusals: null, or what is wrong ---------------------------------------------------------------------------------------------
inline bool paged_aligned(const void *p, uint64_t stride_bytes) { return ((uintptr_t)p | stride_bytes) % 16 == 0; }
inline uint32_t float_bytes(uint32_t type) { return type == LV_F32 ? 4 : type == LV_F16 || type == LV_BF16 ? 2 : 0; }

inline const char *paged_cache_refusal(const lv_paged_cache *c)
{
    if (!c) return "the cache is null";
    if (c->type != LV_F16 && c->type != LV_BF16 && c->type != LV_Q8_0 && c->type != LV_Q4_0) return "the cache's type is none of LV_F16, LV_BF16, LV_Q8_0, LV_Q4_0";
    if (c->dim != 32 && c->dim != 64 && c->dim != 128 && c->dim != 256) return "the head size is none of 32, 64, 128, 256";
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1))) return "a page's tokens are no power of two from 16 to 1024";
    if (c->kv_heads == 0 || c->kv_heads > 4096) return "kv_heads is not in 1 .. 4096";
    if (c->pages == 0) return "there are no pages";
    return nullptr;
}
inline const char *paged_batch_refusal(const lv_paged_cache *c, const lv_paged_batch *b)
{
    if (!b) return "the batch is null";
    if (!c->data) return "the cache has no data";
    if ((uintptr_t)c->data % 16) return "the cache's data is not aligned to 16 bytes";
    if (b->seqs > 65535) return "more than 65535 sequences";
    if (b->tokens >= (1u << 24)) return "2^24 tokens or more";
    if ((uint64_t)b->table_ld * c->page > (1u << 30)) return "the table covers more than 2^30 positions";
    if (b->seqs && (!b->starts || !b->lens || (!b->table && b->table_ld))) return "starts, lens or table is null";
    if (((uintptr_t)b->starts | (uintptr_t)b->lens | (uintptr_t)b->table) % 4) return "starts, lens or table is not aligned to 4 bytes";
    return nullptr;
}
inline const char *paged_rows_refusal(const lv_paged_cache *c, const lv_paged_batch *b, const void *k, uint32_t ldk, const void *v, uint32_t ldv, uint32_t type)
{
    if (const char *e = paged_cache_refusal(c)) return e;
    if (const char *e = paged_batch_refusal(c, b)) return e;
    const uint32_t size = float_bytes(type);
    if (!size) return "the rows' type is none of LV_F32, LV_F16, LV_BF16";
    if (b->tokens == 0 || b->seqs == 0) return nullptr;
    if (!k || !v) return "k or v is null";
    if (ldk < c->kv_heads * c->dim || ldv < c->kv_heads * c->dim) return "a row is longer than its stride";
    if (!paged_aligned(k, (uint64_t)ldk * size) || !paged_aligned(v, (uint64_t)ldv * size)) return "k or v or a stride is not aligned to 16 bytes";
    return nullptr;
}
inline const char *paged_attn_refusal(const lv_paged_cache *c, const lv_paged_batch *b, const lv_paged_attn_spec *s, uint32_t type)
{
    if (const char *e = paged_cache_refusal(c)) return e;
    if (const char *e = paged_batch_refusal(c, b)) return e;
    if (!s) return "the spec is null";
    if (!float_bytes(type)) return "the type is none of LV_F32, LV_F16, LV_BF16";
    if (s->heads == 0 || s->heads > 65536 || s->heads % c->kv_heads) return "heads is no multiple of kv_heads, or not in 1 .. 65536";
    if (!(s->scale - s->scale == 0)) return "the scale is not finite";
    if ((uintptr_t)s->sinks % 4) return "sinks is not aligned to 4 bytes";
    return nullptr;
}
inline const char *paged_attn_rows_refusal(const lv_paged_cache *c, const lv_paged_batch *b, const lv_paged_attn_spec *s, uint32_t type, const void *out, uint32_t ldo,
                                           const void *q, uint32_t ldq)
{
    if (const char *e = paged_attn_refusal(c, b, s, type)) return e;
    if (b->tokens == 0 || b->seqs == 0) return nullptr;
    if (!out || !q) return "out or q is null";
    if (ldo < (uint64_t)s->heads * c->dim || ldq < (uint64_t)s->heads * c->dim) return "a row is longer than its stride";
    const uint32_t size = float_bytes(type);
    if (!paged_aligned(out, (uint64_t)ldo * size) || !paged_aligned(q, (uint64_t)ldq * size)) return "out or q or a stride is not aligned to 16 bytes";
    return nullptr;
}
inline const char *rotate_refusal(const void *out, uint32_t ldo, const void *x, uint32_t ldx, uint32_t type, const uint32_t *positions, uint32_t tokens, uint32_t heads,
                                  uint32_t dim, const lv_rotate_spec *s)
{
    const uint32_t size = float_bytes(type);
    if (!s) return "the spec is null";
    if (!size) return "the type is none of LV_F32, LV_F16, LV_BF16";
    if (dim == 0 || dim > 512 || dim % 8) return "dim is no multiple of 8 from 8 to 512";
    if (heads == 0 || heads > 65536) return "heads is not in 1 .. 65536";
    if (tokens >= (1u << 24)) return "2^24 tokens or more";
    if (s->rot_dims % 2 || s->rot_dims > dim) return "rot_dims is odd or larger than dim";
    if (s->flags & ~(uint32_t)(LV_ROTATE_HALVES | LV_ROTATE_PER_AXIS)) return "unknown flags";
    if (!(s->rot_base > 0) || !(s->rot_base - s->rot_base == 0)) return "rot_base is not above 0, or not finite";
    const uint64_t pairs = (uint64_t)s->sections[0] + s->sections[1] + s->sections[2];
    if (pairs && pairs != s->rot_dims / 2) return "the sections do not add up to rot_dims / 2";
    if (tokens == 0) return nullptr;
    if (!out || !x || !positions) return "out, x or positions is null";
    if ((uint64_t)ldx < (uint64_t)heads * dim || (uint64_t)ldo < (uint64_t)heads * dim) return "a row is longer than its stride";
    if (!paged_aligned(out, (uint64_t)ldo * size) || !paged_aligned(x, (uint64_t)ldx * size)) return "out or x or a stride is not aligned to 16 bytes";
    if ((uintptr_t)positions % 4) return "positions is not aligned to 4 bytes";
    if (out == x && ldo != ldx) return "out is x with another stride";
    return nullptr;
}
inline const char *draft_refusal(const lv_draft_batch *b)
{
    if (!b) return "the batch is null";
    if (b->seqs > 65535) return "more than 65535 sequences";
    if (b->drafts == 0 || b->drafts > 64) return "drafts is not in 1 .. 64";
    if (b->vocab == 0 || b->vocab > (1u << 24)) return "vocab is not in 1 .. 2^24";
    if (b->ld_target < b->vocab || (b->draft && b->ld_draft < b->vocab)) return "a row is longer than its stride";
    if (b->seqs == 0) return nullptr;
    if (!b->target || !b->tokens || !b->uniforms) return "target, tokens or uniforms is null";
    if (((uintptr_t)b->target | (uintptr_t)b->draft | (uintptr_t)b->tokens | (uintptr_t)b->counts | (uintptr_t)b->uniforms) % 4) return "an array is not aligned to 4 bytes";
    return nullptr;
}

}  // namespace lv
