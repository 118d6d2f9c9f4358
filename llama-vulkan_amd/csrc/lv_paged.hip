// lv_paged.hip — lv_kernel_paged_attention: which kernel a call takes, and its launches.
#include <cmath>

#include "lv_paged.h"
#include "lv_serve_host.h"

using namespace lv;

namespace {

struct AttnPlan {
    PagedAttnArgs args{};
    uint32_t tiles;                  // of 16 rows a workgroup; 8: the kernel for tiles
    uint32_t pieces;                 // of a query
    uint64_t items, part_floats, bytes;
};

// Workgroups a compute unit that share the work of a call (lv_paged_plan.h)
constexpr uint32_t kTargetPerUnit = 2;
// The kernel for tiles takes calls whose sequences have more rows than these in the mean, one kernel for all of them: in the mean of all rows of the tensors, those behind the last
// sequence too, over all sequences, those without new tokens too, since the host knows no others (rows of a sequence and key head: new tokens times the heads that share it).  us, rows kernel and
// tiles, 16 sequences of 3000 keys, 8 key heads of 128: fp16 32 rows 39 40, 40 rows 45 41, 64 rows 47 44, 128 rows 65 51; 8 bits 40 rows 50 52, 64 rows 51 55, 80 rows 79 58
constexpr uint32_t kTileRows = 32, kTileRowsBlocks = 64;
// Rows from which the second launch has a wave for each instead of four.
constexpr uint32_t kJoinRows = 1024;
// Calls that are not cut, which saves the second launch and the parts' way through memory: those whose table covers no more positions than these (us, cut and not: one token
// behind 383, 32 heads over 8 of 128 in fp16 11.6 8.9, over 32 11.6 9.0; 256 tokens of 32-bit queries 26.4 14.6; behind 400 32-bit queries over 4-bit rows 12.3 15.3) ...
constexpr uint32_t kWholeKeys = 384;
// ... and chunks, where half of the compute units have a workgroup, whose tiles walk fewer than one and a half times these steps (us, steps of 2 and of 9 at least, fp16: 512
// tokens over 32 key heads 33 20, 1024 over 8 44 29, 1000 behind 500 52 41; 512 behind 1536 42 42, and 53 with steps of 12).
constexpr uint32_t kTileRun = 9;
// Where every compute unit has a workgroup without a cut, sequences are cut for evenness only: into more workgroups than are there at once, which follow as others end, and
// of many steps.  us, 2 a unit of one step at least, 6 of 8, 6 of 16: 64 sequences of 4096 .. 8190 keys, 8 heads of 8 bits 184 174 174; 128 of 1000 .. 2000 of 8 heads in fp16
// 147 153 143; 32 of 2000 .. 4000 84 80 89; 16 of 1000 .. 2000 of 32 heads 80 83 77; 8 of 511 of 32 heads 19.5 15.4 15.4.
constexpr uint32_t kManyPerUnit = 6, kManyRun = 8, kManyMoreRun = 16;

AttnPlan attn_plan(uint32_t units, uint32_t type, const lv_paged_cache &c, const lv_paged_batch &b, const lv_paged_attn_spec &s)
{
    AttnPlan p;
    PagedDeal &d = p.args.deal;
    const uint32_t group = s.heads / c.kv_heads;
    const uint64_t mean = (uint64_t)b.tokens * group / b.seqs;      // rows of a sequence and key head
    p.pieces = type == LV_F32 ? (c.type == LV_BF16 ? 3 : 2) : type == LV_F16 && c.type == LV_BF16 ? 3 : 1;
    const bool blocks = c.type == LV_Q8_0 || c.type == LV_Q4_0;
    const bool tile = p.pieces == 1 && (c.dim == 64 || c.dim == 128) && mean > (blocks ? kTileRowsBlocks : kTileRows);
    p.tiles = tile ? 8 : c.dim <= 128 && mean > 16 ? 2 : 1;      // of 16 rows: keys are read once for each 32 rows where a sequence has more than 16
    d.seqs = b.seqs;
    d.tokens = b.tokens;
    d.group = group;
    d.tile = 16 * p.tiles;
    d.tile_log2 = tile ? 7 : p.tiles == 2 ? 5 : 4;
    d.kv_heads = c.kv_heads;
    d.window = s.window;
    d.chunk = s.chunk;
    d.positions = b.table_ld * c.page;
    d.target = kTargetPerUnit * units;
    const uint64_t whole = (uint64_t)b.tokens * group / d.tile * c.kv_heads;      // workgroups if nothing is cut
    const uint64_t least = (uint64_t)std::min(b.seqs, b.tokens) * c.kv_heads;     // sequences' key heads with something to do, if all have
    d.run_min = tile && whole >= units / 2 ? kTileRun : 1;
    if (!tile && least >= units) {
        d.target = kManyPerUnit * units;
        d.run_min = least >= 2 * units ? kManyMoreRun : kManyRun;
    }
    PagedSeq longest{};
    longest.keys = d.positions;
    if (whole >= d.target || d.positions <= kWholeKeys || paged_parts(paged_steps(d, longest), d.run_min) == 1) d.target = 0;
    p.args.round = units / c.kv_heads;
    p.items = paged_items(d);
    p.part_floats = d.target ? p.items * c.kv_heads * d.tile * c.dim : 0;
    p.bytes = d.target ? (p.part_floats + p.items * c.kv_heads * d.tile * 2) * 4 : 0;
    return p;
}

template <int D, int CT, int NQ, bool FINE = false>
void launch_rows(const AttnPlan &p, uint32_t grid, hipStream_t st)
{
    if constexpr (D <= 128) {
        if (p.tiles == 2) {
            paged_rows_kernel<D, CT, NQ, 2, FINE><<<dim3(grid), dim3(256), 0, st>>>(p.args);
            return;
        }
    }
    paged_rows_kernel<D, CT, NQ, 1, FINE><<<dim3(grid), dim3(256), 0, st>>>(p.args);
}

template <int D, int CT, bool FINE>
void launch_tiles(const PagedAttnArgs &a, uint32_t grid, hipStream_t st) { paged_tile_kernel<D, CT, FINE><<<dim3(grid), dim3(256), 0, st>>>(a); }

template <int D>
void launch_attention(const AttnPlan &p, uint32_t grid, hipStream_t st)
{
    const PagedAttnArgs &a = p.args;
    const bool bf = a.c.type == LV_BF16, fine = a.type == LV_F16;
    float lift = bf ? 0.f : 12.f;
    if (p.tiles == 8) {
        lift = paged_tile_lift(bf);
        if constexpr (D == 64 || D == 128) {
            switch (a.c.type) {
            case LV_F16: launch_tiles<D, kPgF16, false>(a, grid, st); break;
            case LV_BF16: launch_tiles<D, kPgBf16, false>(a, grid, st); break;
            case LV_Q8_0: fine ? launch_tiles<D, kPgQ8, true>(a, grid, st) : launch_tiles<D, kPgQ8, false>(a, grid, st); break;
            default: fine ? launch_tiles<D, kPgQ4, true>(a, grid, st) : launch_tiles<D, kPgQ4, false>(a, grid, st); break;
            }
        }
    } else switch (a.c.type) {
    case LV_F16: p.pieces == 1 ? launch_rows<D, kPgF16, 1>(p, grid, st) : launch_rows<D, kPgF16, 2>(p, grid, st); break;
    case LV_BF16: p.pieces == 1 ? launch_rows<D, kPgBf16, 1>(p, grid, st) : launch_rows<D, kPgBf16, 3>(p, grid, st); break;
    case LV_Q8_0: p.pieces == 1 ? (fine ? launch_rows<D, kPgQ8, 1, true>(p, grid, st) : launch_rows<D, kPgQ8, 1>(p, grid, st)) : launch_rows<D, kPgQ8, 2>(p, grid, st); break;
    default: p.pieces == 1 ? (fine ? launch_rows<D, kPgQ4, 1, true>(p, grid, st) : launch_rows<D, kPgQ4, 1>(p, grid, st)) : launch_rows<D, kPgQ4, 2>(p, grid, st); break;
    }
    if (!a.deal.target) return;
    const uint32_t rows = a.deal.tokens * a.deal.group * a.deal.kv_heads;
    if (rows >= kJoinRows) paged_join_kernel<D, 1><<<dim3((rows + 3) / 4), dim3(256), 0, st>>>(a, lift);
    else paged_join_kernel<D, 4><<<dim3(rows), dim3(256), 0, st>>>(a, lift);
}

}  // namespace

extern "C" int lv_paged_attention_workspace(lv_ctx *c, uint32_t type, const lv_paged_cache *cache, const lv_paged_batch *batch, const lv_paged_attn_spec *spec,
                                            uint64_t *bytes)
{
    if (!bytes) return fail(LV_ERR_ARG, "lv_paged_attention_workspace: bytes is null");
    *bytes = 0;
    if (const char *e = paged_attn_refusal(cache, batch, spec, type)) return fail(LV_ERR_ARG, "lv_paged_attention_workspace: %s", e);
    if (!c) return fail(LV_ERR_ARG, "lv_paged_attention_workspace: ctx is null");
    if (batch->seqs && batch->tokens) *bytes = attn_plan(ctx_units(c), type, *cache, *batch, *spec).bytes;
    return LV_OK;
}

extern "C" int lv_kernel_paged_attention(lv_ctx *c, void *out, uint32_t ldo, const void *q, uint32_t ldq, uint32_t type, const lv_paged_cache *cache,
                                         const lv_paged_batch *batch, const lv_paged_attn_spec *spec, void *work, uint64_t work_bytes)
{
    if (const char *e = paged_attn_rows_refusal(cache, batch, spec, type, out, ldo, q, ldq)) return fail(LV_ERR_ARG, "lv_kernel_paged_attention: %s", e);
    if (!c) return fail(LV_ERR_ARG, "lv_kernel_paged_attention: ctx is null");
    if (batch->seqs == 0 || batch->tokens == 0) return LV_OK;
    AttnPlan p = attn_plan(ctx_units(c), type, *cache, *batch, *spec);
    if (p.bytes && (!work || work_bytes < p.bytes || (uintptr_t)work % 16))
        return fail(LV_ERR_ARG, "lv_kernel_paged_attention: a workspace of %llu bytes, aligned to 16, is needed", (unsigned long long)p.bytes);
    const uint64_t grid = p.items * cache->kv_heads, rows = (uint64_t)batch->tokens * spec->heads;
    // 2^24 workgroups of 256 are more than a launch may have
    if (grid > 0xffffffu || rows > 0x7fffffffu) return fail(LV_ERR_RANGE, "lv_kernel_paged_attention: %u tokens of %u heads", batch->tokens, spec->heads);
    PagedAttnArgs &a = p.args;
    a.c = paged_view(*cache);
    a.starts = batch->starts;
    a.lens = batch->lens;
    a.table = batch->table;
    a.table_ld = batch->table_ld;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.type = type;
    a.scale = spec->scale * 1.44269504088896341f;
    a.sinks = spec->sinks;
    a.items = (uint32_t)p.items;
    a.part = static_cast<float *>(work);
    a.part_ml = a.part + p.part_floats;
    DeviceScope scope(ctx_device(c));
    HIP_TRY(scope.error);
    const hipStream_t st = ctx_stream(c);
    switch (cache->dim) {
    case 32: launch_attention<32>(p, (uint32_t)grid, st); break;
    case 64: launch_attention<64>(p, (uint32_t)grid, st); break;
    case 128: launch_attention<128>(p, (uint32_t)grid, st); break;
    default: launch_attention<256>(p, (uint32_t)grid, st); break;
    }
    HIP_TRY(hipGetLastError());
    return LV_OK;
}
