// lv_serve.hip — entry points of a serving step: rotary positions, rows to and from a paged cache, verification of drafts.
#include <algorithm>
#include <cmath>

#include "lv_serve.h"
#include "lv_serve_host.h"

using namespace lv;

extern "C" int lv_kernel_rotate(lv_ctx *c, void *out, uint32_t ldo, const void *x, uint32_t ldx, uint32_t type, const uint32_t *positions, uint32_t tokens, uint32_t heads,
                                uint32_t dim, const lv_rotate_spec *spec)
{
    if (const char *e = rotate_refusal(out, ldo, x, ldx, type, positions, tokens, heads, dim, spec)) return fail(LV_ERR_ARG, "lv_kernel_rotate: %s", e);
    if (!c) return fail(LV_ERR_ARG, "lv_kernel_rotate: ctx is null");
    if (tokens == 0) return LV_OK;
    const uint32_t half = spec->rot_dims / 2;
    RotateArgs a{};
    a.x = x;
    a.out = out;
    a.positions = positions;
    a.ldx = ldx;
    a.ldo = ldo;
    a.type = type;
    a.tokens = tokens;
    a.heads = heads;
    a.dim = dim;
    a.rot = spec->rot_dims;
    a.flags = spec->flags;
    const bool one = spec->sections[0] + spec->sections[1] + spec->sections[2] == 0;
    const uint32_t sections[3] = {one ? half : spec->sections[0], one ? 0 : spec->sections[1], one ? 0 : spec->sections[2]};
    a.ends[0] = sections[0];
    a.ends[1] = sections[0] + sections[1];
    const double octaves = std::log2(spec->rot_base);
    const bool per_axis = spec->flags & LV_ROTATE_PER_AXIS;
    for (int i = 0; i < 3; i++) {
        const uint32_t pairs = per_axis ? sections[i] : half;
        a.step[i] = pairs ? -octaves / pairs : 0.0;
        a.first[i] = per_axis && i ? a.ends[i - 1] : 0;
    }
    const bool halves = spec->flags & LV_ROTATE_HALVES, vec = spec->rot_dims % (halves ? 16 : 8) == 0;
    const uint32_t units = vec ? spec->rot_dims / (halves ? 16 : 8) + (dim - spec->rot_dims) / 8 : half + dim - spec->rot_dims;
    // Few tokens: a workgroup for every 256 units; many: a few rounds of units share a token's angles
    const uint32_t blocks = (uint32_t)(((uint64_t)heads * units + 255) / 256), y = std::max(1u, std::min(std::min(blocks, 65535u), 2048u / tokens));
    DeviceScope scope(ctx_device(c));
    HIP_TRY(scope.error);
    const hipStream_t st = ctx_stream(c);
    const dim3 grid(tokens, y);
    if (halves && vec) rotate_kernel<true, true><<<grid, dim3(256), 0, st>>>(a);
    else if (halves) rotate_kernel<true, false><<<grid, dim3(256), 0, st>>>(a);
    else if (vec) rotate_kernel<false, true><<<grid, dim3(256), 0, st>>>(a);
    else rotate_kernel<false, false><<<grid, dim3(256), 0, st>>>(a);
    HIP_TRY(hipGetLastError());
    return LV_OK;
}

extern "C" int lv_paged_cache_bytes(const lv_paged_cache *cache, uint64_t *bytes)
{
    if (!bytes) return fail(LV_ERR_ARG, "lv_paged_cache_bytes: bytes is null");
    *bytes = 0;
    if (const char *e = paged_cache_refusal(cache)) return fail(LV_ERR_ARG, "lv_paged_cache_bytes: %s", e);
    *bytes = (uint64_t)cache->pages * cache->kv_heads * paged_view(*cache).block;
    return LV_OK;
}

static int paged_copy(const char *name, bool write, lv_ctx *c, const lv_paged_cache *cache, const lv_paged_batch *batch, void *k, uint32_t ldk, void *v, uint32_t ldv, uint32_t type)
{
    if (const char *e = paged_rows_refusal(cache, batch, k, ldk, v, ldv, type)) return fail(LV_ERR_ARG, "%s: %s", name, e);
    if (!c) return fail(LV_ERR_ARG, "%s: ctx is null", name);
    if (batch->tokens == 0 || batch->seqs == 0) return LV_OK;
    PagedRowsArgs a{};
    a.c = paged_view(*cache);
    a.starts = batch->starts;
    a.lens = batch->lens;
    a.table = batch->table;
    a.seqs = batch->seqs;
    a.tokens = batch->tokens;
    a.table_ld = batch->table_ld;
    a.positions = batch->table_ld * cache->page;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.type = type;
    DeviceScope scope(ctx_device(c));
    HIP_TRY(scope.error);
    // tokens a workgroup: as many as 1024 units hold, but no fewer workgroups than there are compute units
    const uint32_t units = 2 * cache->kv_heads * (cache->dim / 8), room = std::max(1u, std::min(kCopyRun, 256 * kCopyUnits / units));
    const uint32_t run = std::max(1u, std::min(room, batch->tokens / ctx_units(c)));
    const dim3 grid((batch->tokens + run - 1) / run, (units + 256 * kCopyUnits - 1) / (256 * kCopyUnits));
    if (write) paged_copy_kernel<true><<<grid, dim3(256), 0, ctx_stream(c)>>>(a, run);
    else paged_copy_kernel<false><<<grid, dim3(256), 0, ctx_stream(c)>>>(a, run);
    HIP_TRY(hipGetLastError());
    return LV_OK;
}

extern "C" int lv_kernel_paged_write(lv_ctx *c, const lv_paged_cache *cache, const lv_paged_batch *batch, const void *k, uint32_t ldk, const void *v, uint32_t ldv, uint32_t type)
{
    return paged_copy("lv_kernel_paged_write", true, c, cache, batch, const_cast<void *>(k), ldk, const_cast<void *>(v), ldv, type);
}

extern "C" int lv_kernel_paged_read(lv_ctx *c, const lv_paged_cache *cache, const lv_paged_batch *batch, void *k, uint32_t ldk, void *v, uint32_t ldv, uint32_t type)
{
    return paged_copy("lv_kernel_paged_read", false, c, cache, batch, k, ldk, v, ldv, type);
}

// Few and short rows are one launch, a workgroup a sequence.  us, one launch and two, of 1, 16 and 48 sequences: 8192 entries 8.1 11.2, 8.1 11.1, 8.1 11.1; 32000 9.8 11.3,
// 10.1 11.0, 11.8 11.1; 50000 12.4 11.1, 15.8 11.1, 16.6 11.2
static bool verify_one(const lv_draft_batch &b) { return (b.vocab <= 16384 && b.seqs <= 256) || (b.vocab <= 32768 && b.seqs <= 16); }

// entries of a segment, and segments
static void verify_segments(const lv_draft_batch &b, uint32_t &length, uint32_t &segments)
{
    segments = verify_one(b) ? 16 : std::min(kVerifySegments, (b.vocab + kVerifySegment - 1) / kVerifySegment);
    length = ((b.vocab + segments - 1) / segments + 255) / 256 * 256;
    segments = (b.vocab + length - 1) / length;
}
static uint64_t verify_bytes(const lv_draft_batch &b, uint32_t segments) { return verify_one(b) ? 0 : (uint64_t)b.seqs * segments * 2 * sizeof(double); }

extern "C" int lv_verify_drafts_workspace(lv_ctx *c, const lv_draft_batch *batch, uint64_t *bytes)
{
    if (!bytes) return fail(LV_ERR_ARG, "lv_verify_drafts_workspace: bytes is null");
    *bytes = 0;
    if (const char *e = draft_refusal(batch)) return fail(LV_ERR_ARG, "lv_verify_drafts_workspace: %s", e);
    if (!c) return fail(LV_ERR_ARG, "lv_verify_drafts_workspace: ctx is null");
    uint32_t length, segments;
    verify_segments(*batch, length, segments);
    *bytes = verify_bytes(*batch, segments);
    return LV_OK;
}

extern "C" int lv_kernel_verify_drafts(lv_ctx *c, uint32_t *tokens, uint32_t *accepted, const lv_draft_batch *batch, void *work, uint64_t work_bytes)
{
    if (const char *e = draft_refusal(batch)) return fail(LV_ERR_ARG, "lv_kernel_verify_drafts: %s", e);
    if (!c) return fail(LV_ERR_ARG, "lv_kernel_verify_drafts: ctx is null");
    if (batch->seqs == 0) return LV_OK;
    if (!tokens || !accepted || ((uintptr_t)tokens | (uintptr_t)accepted) % 4) return fail(LV_ERR_ARG, "lv_kernel_verify_drafts: tokens or accepted is null or not aligned to 4 bytes");
    VerifyArgs a{};
    a.b = *batch;
    a.tokens = tokens;
    a.accepted = accepted;
    verify_segments(*batch, a.length, a.segments);
    const uint64_t bytes = verify_bytes(*batch, a.segments);
    if (bytes && (!work || work_bytes < bytes || (uintptr_t)work % 16))
        return fail(LV_ERR_ARG, "lv_kernel_verify_drafts: a workspace of %llu bytes, aligned to 16, is needed", (unsigned long long)bytes);
    a.sums = static_cast<double *>(work);
    DeviceScope scope(ctx_device(c));
    HIP_TRY(scope.error);
    const hipStream_t st = ctx_stream(c);
    if (!bytes) {
        verify_whole_kernel<<<dim3(batch->seqs), dim3(1024), 0, st>>>(a);
    } else {
        verify_sums_kernel<<<dim3(a.segments, batch->seqs), dim3(256), 0, st>>>(a);
        verify_pick_kernel<<<dim3(batch->seqs), dim3(256), 0, st>>>(a);
    }
    HIP_TRY(hipGetLastError());
    return LV_OK;
}
