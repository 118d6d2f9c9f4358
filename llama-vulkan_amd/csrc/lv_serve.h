// lv_serve.h — the smaller operators of a serving step: rotary positions, rows to and from a paged cache, verification of drafts.
#pragma once

#include "lv_paged.h"

namespace lv {

// ---- rotary positions --------------------------------------------------------------------------------------------------------------
// A workgroup turns some heads of one token: the angles are the same for all heads, so they are formed once (in turns, in double, reduced to half a turn before
// they become fp32: a position of 10^5 leaves nothing of a 32-bit angle) and read from LDS by every head.  Bound by the bytes of x and out.
struct RotateArgs {
    const void *x;
    void *out;
    const uint32_t *positions;
    uint32_t ldx, ldo, type, tokens, heads, dim, rot, flags;
    uint32_t ends[2];              // pairs of the first axis, and of the first two
    double step[3];                // log2 of the factor from one pair to the next, by axis
    uint32_t first[3];             // pair whose factor is 1, by axis
};

// VEC: units of 8 elements (pairs of neighbours), or 8 and their 8 partners; otherwise a unit is a pair.  Behind them units of 8 or 1 that are copied.
template <bool HALVES, bool VEC>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a)
{
    __shared__ float2 turn[256];
    const uint32_t token = blockIdx.x, half = a.rot / 2;
    for (uint32_t i = threadIdx.x; i < half; i += 256) {
        const uint32_t axis = i < a.ends[0] ? 0 : i < a.ends[1] ? 1 : 2;
        const double f = (double)a.positions[(uint64_t)axis * a.tokens + token] * (exp2((double)(i - a.first[axis]) * a.step[axis]) * 0.15915494309189533577);
        float s, c;
        sincospif(2.f * (float)(f - rint(f)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    const uint32_t turned = VEC ? a.rot / (HALVES ? 16 : 8) : half, units = turned + (VEC ? (a.dim - a.rot) / 8 : a.dim - a.rot);
    const uint64_t from = (uint64_t)token * a.ldx, to = (uint64_t)token * a.ldo;
    for (uint32_t n = blockIdx.y * 256 + threadIdx.x; n < a.heads * units; n += gridDim.y * 256) {
        const uint32_t h = n / units, u = n - h * units, at = h * a.dim;
        if constexpr (VEC) {
            float p[8], q[8];
            if (u >= turned) {
                if (a.out == a.x) continue;
                const uint32_t d = at + a.rot + (u - turned) * 8;
                pg_load8(a.x, a.type, from + d, p);
                pg_store8(a.out, a.type, to + d, p);
            } else if constexpr (HALVES) {
                pg_load8(a.x, a.type, from + at + u * 8, p);
                pg_load8(a.x, a.type, from + at + half + u * 8, q);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float2 t = turn[u * 8 + e];
                    const float v = p[e] * t.x - q[e] * t.y;
                    q[e] = p[e] * t.y + q[e] * t.x;
                    p[e] = v;
                }
                pg_store8(a.out, a.type, to + at + u * 8, p);
                pg_store8(a.out, a.type, to + at + half + u * 8, q);
            } else {
                pg_load8(a.x, a.type, from + at + u * 8, p);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 t = turn[u * 4 + e];
                    const float v = p[2 * e] * t.x - p[2 * e + 1] * t.y;
                    p[2 * e + 1] = p[2 * e] * t.y + p[2 * e + 1] * t.x;
                    p[2 * e] = v;
                }
                pg_store8(a.out, a.type, to + at + u * 8, p);
            }
        } else {
            auto get = [&](uint64_t i) {
                if (a.type == LV_F32) return static_cast<const float *>(a.x)[i];
                const uint16_t v = static_cast<const uint16_t *>(a.x)[i];
                return a.type == LV_F16 ? half_bits_to_float(v) : __uint_as_float((uint32_t)v << 16);
            };
            auto set = [&](uint64_t i, float v) {
                if (a.type == LV_F32) static_cast<float *>(a.out)[i] = v;
                else static_cast<uint16_t *>(a.out)[i] = (uint16_t)pg_bits(v, a.type == LV_F16);
            };
            if (u >= turned) {
                if (a.out != a.x) set(to + at + a.rot + u - turned, get(from + at + a.rot + u - turned));
                continue;
            }
            const uint32_t i = HALVES ? u : 2 * u, j = HALVES ? u + half : 2 * u + 1;
            const float2 t = turn[u];
            const float p = get(from + at + i), q = get(from + at + j);
            set(to + at + i, p * t.x - q * t.y);
            set(to + at + j, p * t.y + q * t.x);
        }
    }
}

// ---- rows to pages and back ----------------------------------------------------------------------------------------------------------
struct PagedRowsArgs {
    PagedView c;
    const uint32_t *starts, *lens, *table;
    uint32_t seqs, tokens, table_ld, positions;
    void *k, *v;
    uint32_t ldk, ldv, type;
};

// where a row's token lies: the page, or kNoPage, and the place in it.  By every wave on its own; `row` is the same in all lanes
__device__ __forceinline__ uint32_t paged_place(const PagedRowsArgs &a, uint32_t row, uint32_t &in)
{
    const int lane = threadIdx.x & 63;
    for (uint32_t b0 = 0; b0 < a.seqs; b0 += 64) {
        PagedSeq s{};
        uint32_t page = kNoPage, at = 0;
        if (b0 + lane < a.seqs) s = paged_seq(a.starts[b0 + lane], a.starts[b0 + lane + 1], a.lens[b0 + lane], a.tokens, a.positions);
        const bool mine = row >= s.row0 && row - s.row0 < s.rows;
        if (mine) {
            const int32_t p = s.pos0 + (int32_t)(row - s.row0);
            if (p >= 0) {
                page = paged_page(a.c, a.table + (uint64_t)(b0 + lane) * a.table_ld, a.table_ld, (uint32_t)p);
                at = (uint32_t)p & ((1u << a.c.shift) - 1);
            }
        }
        const uint64_t here = __ballot(mine);
        if (here) {
            const int l = __builtin_ctzll(here);
            in = __builtin_amdgcn_readlane(at, l);
            return __builtin_amdgcn_readlane(page, l);
        }
    }
    return kNoPage;
}

// A thread takes eight elements, four neighbouring threads a block of 32.  grid (tokens, units / 256).  Bound by the bytes of the rows.
template <bool WRITE>
__global__ __launch_bounds__(256) void paged_copy_kernel(PagedRowsArgs a)
{
    const uint32_t per = a.c.dim / 8, units = 2 * a.c.kv_heads * per, u = blockIdx.y * 256 + threadIdx.x, row = blockIdx.x;
    const bool mine = u < units;
    const uint32_t which = u >= units / 2 ? 1 : 0, w = u - which * (units / 2), head = w / per, d = (w - head * per) * 8;
    const uint64_t at = (uint64_t)row * (which ? a.ldv : a.ldk) + (uint64_t)w * 8;
    void *rows = which ? a.v : a.k;
    float x[8];
    if (WRITE && mine) pg_load8(rows, a.type, at, x);      // on its way while the page is looked up
    uint32_t in = 0;
    const uint32_t page = paged_place(a, row, in);
    if (page == kNoPage || !mine) return;      // whole groups of four: units is a multiple of 8
    uint8_t *codes = a.c.data + paged_codes(a.c, page, head, which, in), *scales = a.c.data + paged_scales(a.c, page, head, which, in);
    if (a.c.type == LV_F16 || a.c.type == LV_BF16) {
        if constexpr (WRITE) {
            pg_store8(codes, a.c.type, d, x);
        } else {
            pg_load8(codes, a.c.type, d, x);
            pg_store8(rows, a.type, at, x);
        }
        return;
    }
    const bool eight = a.c.type == LV_Q8_0;
    uint16_t *scale = reinterpret_cast<uint16_t *>(scales) + d / 32;
    const uint32_t quarter = d / 8 % 4;      // of the block
    if constexpr (WRITE) {
        float hi = -INFINITY, lo = INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            hi = fmaxf(hi, x[e]);      // of a number and NaN, the number
            lo = fminf(lo, x[e]);
        }
        hi = fmaxf(hi, dpp_mov<0xB1>(hi));
        hi = fmaxf(hi, dpp_mov<0x4E>(hi));
        lo = fminf(lo, dpp_mov<0xB1>(lo));
        lo = fminf(lo, dpp_mov<0x4E>(lo));
        if (hi < lo) hi = lo = 0.f;      // nothing but NaN
        float s;
        if (eight) s = fminf(fmaxf(hi, -lo) * (1.f / 127.f), 515.5f);
        else s = fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -8188.f), 8188.f);
        uint16_t h = float_to_half_bits(s);
        if ((h & 0x7fffu) == 0) h = 0;
        const float back = half_bits_to_float(h), inv = back == 0.f ? 0.f : 1.f / back;
        int q[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float c = rintf(x[e] * inv);
            q[e] = x[e] == x[e] && inv != 0.f ? (int)fminf(fmaxf(c, eight ? -127.f : -8.f), eight ? 127.f : 7.f) : 0;
        }
        if (quarter == 0) *scale = h;
        if (eight) {
            uint32_t lo4 = 0, hi4 = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo4 |= ((uint32_t)q[e] & 0xffu) << (8 * e);
                hi4 |= ((uint32_t)q[4 + e] & 0xffu) << (8 * e);
            }
            *reinterpret_cast<uint2 *>(codes + d) = make_uint2(lo4, hi4);
        } else {
            uint32_t lo4 = 0, hi4 = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo4 |= ((uint32_t)(q[e] + 8) & 0xfu) << (8 * e);
                hi4 |= ((uint32_t)(q[4 + e] + 8) & 0xfu) << (8 * e);
            }
            // lanes 0 and 1 of four hold elements 0 .. 15 and get 16 .. 31 from lanes 2 and 3
            const uint32_t up_lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo4, 0xEE, 0xf, 0xf, true);
            const uint32_t up_hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi4, 0xEE, 0xf, 0xf, true);
            if (quarter < 2) *reinterpret_cast<uint2 *>(codes + d / 32 * 16 + quarter * 8) = make_uint2(lo4 | (up_lo << 4), hi4 | (up_hi << 4));
        }
    } else {
        const float s = half_bits_to_float(*scale);
        if (eight) {
            const uint2 q = *reinterpret_cast<const uint2 *>(codes + d);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = s * (float)(int8_t)((e < 4 ? q.x : q.y) >> (8 * (e % 4)));
        } else {
            const uint2 q = *reinterpret_cast<const uint2 *>(codes + d / 32 * 16 + quarter % 2 * 8);
            const int shift = quarter < 2 ? 0 : 4;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = s * (float)((int)(((e < 4 ? q.x : q.y) >> (8 * (e % 4) + shift)) & 0xfu) - 8);
        }
        pg_store8(rows, a.type, at, x);
    }
}

// ---- verification of drafts ------------------------------------------------------------------------------------------------------------
// Two launches: the weights' sums over segments of the row that decides, many workgroups a sequence; then the segment that the random number falls into,
// a workgroup a sequence.  Sums in double: a running sum of 10^5 floats in 32 bits is off by more than the smallest probabilities.
struct VerifyArgs {
    lv_draft_batch b;
    uint32_t *tokens, *accepted;
    double *sums;              // [seqs][segments][2]: what is left of the target after the draft, and the target
    uint32_t segments, length; // entries of a segment, a multiple of 256
};
constexpr uint32_t kVerifySegment = 2048, kVerifySegments = 64;

// the drafts of sequence b that stand, and how many there are; by every wave on its own
__device__ __forceinline__ uint32_t verify_standing(const lv_draft_batch &b, uint32_t seq, uint32_t &count)
{
    const uint32_t i = threadIdx.x & 63;
    count = b.counts ? min(b.counts[seq], b.drafts) : b.drafts;
    bool stands = false;
    if (i < count) {
        const uint32_t x = b.tokens[(uint64_t)seq * b.drafts + i];
        if (x < b.vocab) {
            const float p = b.target[((uint64_t)seq * (b.drafts + 1) + i) * b.ld_target + x], u = b.uniforms[(uint64_t)seq * (b.drafts + 1) + i];
            const float q = b.draft ? b.draft[((uint64_t)seq * b.drafts + i) * b.ld_draft + x] : 1.f;
            stands = (double)u * (double)q < (double)p;
        }
    }
    const uint64_t not_standing = __ballot(!stands);      // 64 drafts that all stand leave none
    return not_standing ? min((uint32_t)__builtin_ctzll(not_standing), count) : count;
}

struct VerifyRow {
    const float *p, *q;        // q null: nothing, or with `x` below vocab the draft was picked and only its own token is taken out
    uint32_t x;
};
__device__ __forceinline__ VerifyRow verify_row(const lv_draft_batch &b, uint32_t seq, uint32_t r, uint32_t count)
{
    VerifyRow v;
    v.p = b.target + ((uint64_t)seq * (b.drafts + 1) + r) * b.ld_target;
    v.q = r < count && b.draft ? b.draft + ((uint64_t)seq * b.drafts + r) * b.ld_draft : nullptr;
    v.x = r < count && !b.draft ? b.tokens[(uint64_t)seq * b.drafts + r] : 0xffffffffu;
    return v;
}
__device__ __forceinline__ double verify_whole(float p) { return p > 0.f ? (double)p : 0.0; }
__device__ __forceinline__ double verify_rest(const VerifyRow &v, uint32_t j, float p, float q)
{
    if (j == v.x) return 0.0;
    const double d = (double)p - (v.q ? (double)q : 0.0);
    return d > 0.0 ? d : 0.0;
}

__device__ __forceinline__ double wave_sum_double(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// grid (segments, seqs)
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a)
{
    __shared__ double part[4][2];
    const uint32_t seq = blockIdx.y, j0 = blockIdx.x * a.length, j1 = min(j0 + a.length, a.b.vocab);
    uint32_t count;
    const uint32_t r = verify_standing(a.b, seq, count);
    const VerifyRow row = verify_row(a.b, seq, r, count);
    double rest = 0.0, whole = 0.0;
    for (uint32_t j = j0 + threadIdx.x; j < j1; j += 256) {
        const float p = row.p[j], q = row.q ? row.q[j] : 0.f;
        rest += verify_rest(row, j, p, q);
        whole += verify_whole(p);
    }
    rest = wave_sum_double(rest);
    whole = wave_sum_double(whole);
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6][0] = rest;
        part[threadIdx.x >> 6][1] = whole;
    }
    __syncthreads();
    if (threadIdx.x < 2) a.sums[((uint64_t)seq * a.segments + blockIdx.x) * 2 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// grid (seqs)
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a)
{
    __shared__ double waves[4];
    __shared__ uint32_t found, last;
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t count;
    const uint32_t r = verify_standing(a.b, seq, count);
    const VerifyRow row = verify_row(a.b, seq, r, count);
    // segments, 64 at most: running sums by lane
    const bool mine = lane < a.segments;
    const double rest = mine ? a.sums[((uint64_t)seq * a.segments + lane) * 2] : 0.0, whole = mine ? a.sums[((uint64_t)seq * a.segments + lane) * 2 + 1] : 0.0;
    const bool use_rest = wave_sum_double(rest) > 0.0;
    double upto = use_rest ? rest : whole;
    const double own = upto;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double v = __shfl_up(upto, off, 64);
        if (lane >= (uint32_t)off) upto += v;
    }
    const double total = __shfl(upto, 63, 64), goal = (double)a.b.uniforms[(uint64_t)seq * (a.b.drafts + 1) + a.b.drafts] * total;
    // the first segment whose running sum is more; where a rounding leaves none, the last that holds something
    const uint64_t over = __ballot(mine && upto > goal), any = __ballot(mine && own > 0.0);
    uint32_t pick = 0;
    if (any) {
        const int seg = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        const double before = __shfl(upto - own, seg, 64);
        const uint32_t j0 = seg * a.length, j1 = min(j0 + a.length, a.b.vocab), each = a.length / 256;
        if (threadIdx.x == 0) {
            found = 0xffffffffu;
            last = 0;
        }
        auto weight = [&](uint32_t j) {
            const float p = row.p[j];
            return use_rest ? verify_rest(row, j, p, row.q ? row.q[j] : 0.f) : verify_whole(p);
        };
        const uint32_t from = j0 + threadIdx.x * each, to = min(from + each, j1);
        double sum = 0.0;
        uint32_t some = 0xffffffffu;
        for (uint32_t j = from; j < to; j++) {
            const double w = weight(j);
            sum += w;
            if (w > 0.0) some = j;
        }
        double run = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double v = __shfl_up(run, off, 64);
            if (lane >= (uint32_t)off) run += v;
        }
        if (lane == 63) waves[wave] = run;
        __syncthreads();
        double start = before;
        for (uint32_t w = 0; w < wave; w++) start += waves[w];
        run += start;
        // the first thread whose sums pass the goal looks for the place; the last one that holds something is the way out
        const bool passes = run > goal && sum > 0.0;
        const uint64_t first = __ballot(passes), holds = __ballot(some != 0xffffffffu);
        if (first && lane == (uint32_t)__builtin_ctzll(first)) {
            double at = run - sum;
            uint32_t j = from;
            uint32_t best = some;
            for (; j < to; j++) {
                const double w = weight(j);
                at += w;
                if (w > 0.0 && at > goal) {
                    best = j;
                    break;
                }
            }
            atomicMin(&found, best);
        }
        if (holds && lane == (uint32_t)(63 - __builtin_clzll(holds))) atomicMax(&last, some);
        __syncthreads();
        pick = found != 0xffffffffu ? found : last;
    }
    if (threadIdx.x <= a.b.drafts && threadIdx.x < 65) {
        const uint32_t i = threadIdx.x;
        a.tokens[(uint64_t)seq * (a.b.drafts + 1) + i] = i < r ? a.b.tokens[(uint64_t)seq * a.b.drafts + i] : i == r ? pick : (uint32_t)LV_NO_TOKEN;
    }
    if (threadIdx.x == 0) a.accepted[seq] = r;
}

}  // namespace lv
