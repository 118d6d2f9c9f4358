// lv_serve.h — the smaller operators of a serving step: rotary positions, rows to and from a paged cache, verification of drafts.
#pragma once

#include "lv_paged.h"

namespace lv {

// ---- rotary positions --------------------------------------------------------------------------------------------------------------
// A workgroup turns some heads of one token: the angles are the same for all heads, so they are formed once (in turns, in double, reduced to half a turn before
// they become fp32: a position of 10^5 leaves nothing of a 32-bit angle) and read from LDS by every head.  Bound by the bytes of x and out
// (6001 tokens of 40 heads of 128, bf16: 21 us, 5.8 TB/s, part of it from the last cache); one token by its launch (2.7).
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

// where the tokens of rows row0 + lane lie: the page, or kNoPage, and the place in it.  By a whole wave; lanes from `rows` on find nothing
__device__ __forceinline__ uint2 paged_places(const PagedRowsArgs &a, uint32_t row0, uint32_t rows, uint32_t lane)
{
    // the last sequence that starts at row0 or before it: 64 at a time; then, where a lane's row is not that sequence's, by halves
    uint32_t first = 0;
    for (uint32_t b0 = 0; b0 < a.seqs; b0 += 64) {
        const uint64_t from_here = __ballot(b0 + lane < a.seqs && a.starts[min(b0 + lane, a.seqs)] <= row0);
        if (from_here) first = b0 + 63 - __builtin_clzll(from_here);
        if (from_here != ~0ull) break;
    }
    uint2 out = make_uint2(kNoPage, 0);
    if (lane >= rows) return out;
    const uint32_t row = row0 + lane;
    uint32_t b = first, n = a.starts[first + 1] <= row ? a.seqs - first : 1;
    while (n > 1) {
        const uint32_t half = n / 2;
        const bool up = a.starts[b + half] <= row;
        b = up ? b + half : b;
        n = up ? n - half : half;
    }
    const PagedSeq s = paged_seq(a.starts[b], a.starts[b + 1], a.lens[b], a.tokens, a.positions);
    if (row < s.row0 || row - s.row0 >= s.rows) return out;
    const int32_t p = s.pos0 + (int32_t)(row - s.row0);
    if (p < 0) return out;
    out.x = paged_page(a.c, a.table + (uint64_t)b * a.table_ld, a.table_ld, (uint32_t)p);
    out.y = (uint32_t)p & ((1u << a.c.shift) - 1);
    return out;
}

// rint(x * inv) between low and high, 0 for NaN, plus magic
__device__ __forceinline__ float paged_code(float x, float inv, float low, float high, float magic)
{
#pragma clang fp contract(off)
    const float c = x * inv;
    return (c == c ? __builtin_amdgcn_fmed3f(c, low, high) : 0.f) + magic;
}

// eight numbers of a block of 32 as it is stored; the block's are in four neighbouring threads, `quarter` says which
__device__ __forceinline__ void paged_put_block(const float (&x)[8], bool eight, uint32_t quarter, uint8_t *block_codes, uint16_t *scale)
{
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
    // A number of up to 2^22 plus 1.5 * 2^23 is rounded to an integer, ties to even, whose low byte is the sum's.  The product is rounded first: no fma.
    const float low = eight ? -127.f : -8.f, high = eight ? 127.f : 7.f, magic = eight ? 12582912.f : 12582920.f;
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; e++) b[e] = __float_as_uint(paged_code(x[e], inv, low, high, magic));
    auto bytes = [](uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c3, c2, 0x0c0c0400u), __builtin_amdgcn_perm(c1, c0, 0x0c0c0400u), 0x05040100u);
    };
    const uint32_t lo4 = bytes(b[0], b[1], b[2], b[3]), hi4 = bytes(b[4], b[5], b[6], b[7]);
    if (quarter == 0) *scale = h;
    if (eight) {
        *reinterpret_cast<uint2 *>(block_codes + quarter * 8) = make_uint2(lo4, hi4);
        return;
    }
    // the first two of four hold elements 0 .. 15 and get 16 .. 31 from the other two
    const uint32_t up_lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo4, 0xEE, 0xf, 0xf, true);
    const uint32_t up_hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi4, 0xEE, 0xf, 0xf, true);
    if (quarter < 2) *reinterpret_cast<uint2 *>(block_codes + quarter * 8) = make_uint2(lo4 | (up_lo << 4), hi4 | (up_hi << 4));
}

// A unit is eight elements of a token's keys or values, four neighbouring threads have a block of 32.  A workgroup takes `run` tokens, up to 1024 units of them, and
// asks for four units a thread before it uses the first: with one token a workgroup the look-up of its page, three loads in a row, was most of a copy's time
// (sequences of 8001 to 16001 tokens of 8 key heads in 8 bits read back: 85 us, and 52, 4.8 TB/s; one unit a thread 95, two 69).  grid (tokens / run, units of a token / 1024).
// Bound by the bytes of the rows, then by the vector work on codes (4095 tokens of 32 heads, 4 bits: written in 45 us, 3.4 TB/s, read back in 29, 5.2).
constexpr uint32_t kCopyUnits = 4, kCopyRun = 64;

// Workgroup i of n as a place in 0 .. n - 1 such that the workgroups of one XCD, every eighth, get neighbouring places: a token's scales, and its codes of 4 bits,
// fill less than a line of the cache, and lines that two XCDs write go to memory twice.
__device__ __forceinline__ uint32_t paged_eighth(uint32_t i, uint32_t n)
{
    const uint32_t x = i % 8, q = n / 8, r = n % 8;
    return x * q + min(x, r) + i / 8;
}

template <bool WRITE>
__global__ __launch_bounds__(256) void paged_copy_kernel(PagedRowsArgs a, uint32_t run)
{
    __shared__ uint2 places[kCopyRun];
    const uint32_t per = a.c.dim / 8, log2_per = 31 - __builtin_clz(per), half = a.c.kv_heads * per, units = 2 * half, row0 = paged_eighth(blockIdx.x, gridDim.x) * run, u0 = blockIdx.y * 256 * kCopyUnits;
    const uint32_t rows = min(run, a.tokens - row0), width = min(units - u0, 256 * kCopyUnits), all = rows * width;      // run is 1 where a token has more units
    const bool blocks = a.c.type == LV_Q8_0 || a.c.type == LV_Q4_0, eight = a.c.type == LV_Q8_0;
    float x[kCopyUnits][8];
    uint32_t row[kCopyUnits], u[kCopyUnits];
    void *rows_at[kCopyUnits];
    uint64_t at[kCopyUnits];
#pragma unroll
    for (uint32_t i = 0; i < kCopyUnits; i++) {
        const uint32_t n = min(i * 256 + threadIdx.x, all - 1);
        row[i] = rows == 1 ? 0 : n / width;
        u[i] = u0 + n - row[i] * width;
        const uint32_t which = u[i] >= half ? 1 : 0;
        rows_at[i] = which ? a.v : a.k;
        at[i] = (uint64_t)(row0 + row[i]) * (which ? a.ldv : a.ldk) + (uint64_t)(u[i] - which * half) * 8;
    }
    if constexpr (WRITE) {
        if (a.type == LV_F32) {
#pragma unroll
            for (uint32_t i = 0; i < kCopyUnits; i++) pg_load8(rows_at[i], LV_F32, at[i], x[i]);
        } else {
            uint4 w[kCopyUnits];
#pragma unroll
            for (uint32_t i = 0; i < kCopyUnits; i++) w[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(rows_at[i]) + at[i]);
#pragma unroll
            for (uint32_t i = 0; i < kCopyUnits; i++) {
                if (a.type == LV_F16) pg_unpack8<false>(w[i], x[i]);
                else pg_unpack8<true>(w[i], x[i]);
            }
        }
    }
    if (threadIdx.x < 64) {
        const uint2 p = paged_places(a, row0, rows, threadIdx.x);
        if (threadIdx.x < rows) places[threadIdx.x] = p;
    }
    __syncthreads();
    uint8_t *codes[kCopyUnits], *scales[kCopyUnits];
    bool mine[kCopyUnits];
    uint32_t d[kCopyUnits];
#pragma unroll
    for (uint32_t i = 0; i < kCopyUnits; i++) {
        const uint2 p = places[row[i]];
        const uint32_t which = u[i] >= half ? 1 : 0, w = u[i] - which * half, head = w >> log2_per;
        d[i] = (w & (per - 1)) * 8;
        mine[i] = i * 256 + threadIdx.x < all && p.x != kNoPage;      // whole groups of four: units and width are multiples of 8
        const uint32_t page = p.x != kNoPage ? p.x : 0;
        codes[i] = a.c.data + paged_codes(a.c, page, head, which, p.y);
        scales[i] = a.c.data + paged_scales(a.c, page, head, which, p.y) + d[i] / 32 * 2;
    }
    if constexpr (WRITE) {
#pragma unroll
        for (uint32_t i = 0; i < kCopyUnits; i++) {
            if (!mine[i]) continue;
            if (blocks) paged_put_block(x[i], eight, d[i] / 8 % 4, codes[i] + d[i] / 32 * (eight ? 32 : 16), reinterpret_cast<uint16_t *>(scales[i]));
            else pg_store8(codes[i], a.c.type, d[i], x[i]);
        }
    } else {
        uint4 w[kCopyUnits];
        uint16_t s[kCopyUnits];
        if (!blocks) {
#pragma unroll
            for (uint32_t i = 0; i < kCopyUnits; i++) w[i] = *reinterpret_cast<const uint4 *>(codes[i] + d[i] * 2);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kCopyUnits; i++) {
                const uint2 q = *reinterpret_cast<const uint2 *>(codes[i] + (eight ? d[i] : d[i] / 32 * 16 + d[i] / 8 % 2 * 8));
                w[i] = make_uint4(q.x, q.y, 0, 0);
                s[i] = *reinterpret_cast<const uint16_t *>(scales[i]);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kCopyUnits; i++) {
            if (!blocks) {
                if (a.c.type == LV_F16) pg_unpack8<false>(w[i], x[i]);
                else pg_unpack8<true>(w[i], x[i]);
            } else {
                // f * (byte - bias) by one rounding: f * bias is exact
                const float f = half_bits_to_float(s[i]), less = -f * (eight ? 128.f : 8.f);
                const uint32_t shift = d[i] / 8 % 4 < 2 ? 0 : 4, flip = eight ? 0x80808080u : 0u, mask = eight ? 0xffffffffu : 0x0f0f0f0fu;
                const uint32_t lo = ((w[i].x ^ flip) >> (eight ? 0 : shift)) & mask, hi = ((w[i].y ^ flip) >> (eight ? 0 : shift)) & mask;
#pragma unroll
                for (int e = 0; e < 8; e++) x[i][e] = fmaf(f, (float)(((e < 4 ? lo : hi) >> (8 * (e % 4))) & 0xffu), less);
            }
            if (mine[i]) pg_store8(rows_at[i], a.type, at[i], x[i]);
        }
    }
}

// ---- verification of drafts ------------------------------------------------------------------------------------------------------------
// Two launches: the weights' sums over segments of the row that decides, many workgroups a sequence; then the segment that the random number falls into,
// a workgroup a sequence (48 sequences, 7 drafts, 128256 entries: 11 us, 4.1 TB/s, and 4.5; segments of 4096 entries a microsecond more in all).  Sums in double: a running sum of 10^5 floats in 32 bits is off by more than the smallest probabilities.
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
    const float *p, *q;        // q null: nothing is taken off but, with `x` below vocab, the one token that was picked
    uint32_t x;
    bool wide;                 // rows of 16-byte alignment
};
__device__ __forceinline__ VerifyRow verify_row(const lv_draft_batch &b, uint32_t seq, uint32_t r, uint32_t count)
{
    VerifyRow v;
    v.p = b.target + ((uint64_t)seq * (b.drafts + 1) + r) * b.ld_target;
    v.q = r < count && b.draft ? b.draft + ((uint64_t)seq * b.drafts + r) * b.ld_draft : nullptr;
    v.x = r < count && !b.draft ? b.tokens[(uint64_t)seq * b.drafts + r] : 0xffffffffu;
    v.wide = ((uintptr_t)v.p | (uintptr_t)v.q) % 16 == 0;
    return v;
}
__device__ __forceinline__ double verify_whole(float p) { return p > 0.f ? (double)p : 0.0; }
__device__ __forceinline__ double verify_rest(uint32_t picked, uint32_t j, float p, float q)
{
    const double d = j == picked ? 0.0 : (double)p - (double)q;
    return d > 0.0 ? d : 0.0;
}
// entries j .. j + 3 of a row, j a multiple of 4; 0 from `end` on
__device__ __forceinline__ void verify_load4(const VerifyRow &v, uint32_t j, uint32_t end, float (&p)[4], float (&q)[4])
{
    if (v.wide && j + 4 <= end) {
        const float4 x = *reinterpret_cast<const float4 *>(v.p + j), y = v.q ? *reinterpret_cast<const float4 *>(v.q + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
        q[0] = y.x; q[1] = y.y; q[2] = y.z; q[3] = y.w;
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        p[e] = j + e < end ? v.p[j + e] : 0.f;
        q[e] = v.q && j + e < end ? v.q[j + e] : 0.f;
    }
}

__device__ __forceinline__ double wave_sum_double(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// what is left of the target after the draft, and the target, summed up by a wave whose lanes take entries j .. j + 3 and so on, `step` further each time; AHEAD of them
// asked for at once
template <int AHEAD> __device__ __forceinline__ void verify_sums(const VerifyRow &row, uint32_t j, uint32_t end, uint32_t step, double &rest, double &whole)
{
    auto add = [&](uint32_t at, const float (&p)[4], const float (&q)[4]) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            rest += verify_rest(row.x, at + e, p[e], q[e]);
            whole += verify_whole(p[e]);
        }
    };
    if (row.wide) {
        for (; j + (AHEAD - 1) * step + 4 <= end; j += AHEAD * step) {
            float p[AHEAD][4], q[AHEAD][4];
#pragma unroll
            for (int n = 0; n < AHEAD; n++) {
                const float4 x = *reinterpret_cast<const float4 *>(row.p + j + n * step), y = row.q ? *reinterpret_cast<const float4 *>(row.q + j + n * step) : make_float4(0.f, 0.f, 0.f, 0.f);
                p[n][0] = x.x; p[n][1] = x.y; p[n][2] = x.z; p[n][3] = x.w;
                q[n][0] = y.x; q[n][1] = y.y; q[n][2] = y.z; q[n][3] = y.w;
            }
#pragma unroll
            for (int n = 0; n < AHEAD; n++) add(j + n * step, p[n], q[n]);
        }
    }
    for (; j < end; j += step) {
        float p[4], q[4];
        verify_load4(row, j, end, p, q);
        add(j, p, q);
    }
    rest = wave_sum_double(rest);
    whole = wave_sum_double(whole);
}

// grid (segments, seqs)
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a)
{
    __shared__ double part[4][2];
    const uint32_t seq = blockIdx.y, j0 = blockIdx.x * a.length, j1 = min(j0 + a.length, a.b.vocab);
    uint32_t count;
    const uint32_t r = verify_standing(a.b, seq, count);
    const VerifyRow row = verify_row(a.b, seq, r, count);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.accepted[seq] = r;
    double rest = 0.0, whole = 0.0;
    verify_sums<2>(row, j0 + 4 * threadIdx.x, j1, 1024, rest, whole);
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6][0] = rest;
        part[threadIdx.x >> 6][1] = whole;
    }
    __syncthreads();
    if (threadIdx.x < 2) a.sums[((uint64_t)seq * a.segments + blockIdx.x) * 2 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// The token of the row, and all tokens of the sequence.  By a workgroup, the first 256 threads of it do the work; rest and whole: the segments' sums, by lane in every wave
__device__ __forceinline__ void verify_pick(const VerifyArgs &a, uint32_t seq, uint32_t r, const VerifyRow &row, double rest, double whole)
{
    __shared__ double waves[4];
    __shared__ uint32_t found, last;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool mine = lane < a.segments, works = threadIdx.x < 256;
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
        double before = __shfl(upto - own, seg, 64);
        const uint32_t j0 = seg * a.length, j1 = min(j0 + a.length, a.b.vocab);
        if (threadIdx.x == 0) {
            found = 0xffffffffu;
            last = 0;
        }
        // 2048 entries at a time, eight neighbours a thread, until the running sum passes the goal; the last entry that holds something is the way out
        for (uint32_t k0 = j0; k0 < j1; k0 += 2048) {
            const uint32_t from = k0 + threadIdx.x * 8;
            double w[8], sum = 0.0;
            uint32_t some = 0xffffffffu;
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                float p[4], q[4];
                verify_load4(row, works ? min(from + 4 * h, j1) : j1, j1, p, q);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) w[4 * h + e] = use_rest ? verify_rest(row.x, from + 4 * h + e, p[e], q[e]) : verify_whole(p[e]);
            }
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) {
                sum += w[e];
                some = w[e] > 0.0 ? from + e : some;
            }
            double run = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const double v = __shfl_up(run, off, 64);
                if (lane >= (uint32_t)off) run += v;
            }
            if (lane == 63 && works) waves[wave] = run;
            __syncthreads();
            double start = before;
            for (uint32_t v = 0; v < min(wave, 4u); v++) start += waves[v];
            const double all = before + ((waves[0] + waves[1]) + (waves[2] + waves[3]));
            run += start;
            const uint64_t first = __ballot((run > goal) & (sum > 0.0)), holds = __ballot(some != 0xffffffffu);
            if (first && lane == (uint32_t)__builtin_ctzll(first)) {
                double at = run - sum;
                uint32_t best = some;
                bool open = true;
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) {
                    at += w[e];
                    const bool here = open & (w[e] > 0.0) & (at > goal);
                    best = here ? from + e : best;
                    open = here ? false : open;
                }
                atomicMin(&found, best);
            }
            if (holds && lane == (uint32_t)(63 - __builtin_clzll(holds))) atomicMax(&last, some);
            __syncthreads();
            before = all;
            if (found != 0xffffffffu) break;      // the same in all threads
            __syncthreads();                      // before `waves` is written again
        }
        pick = found != 0xffffffffu ? found : last;
    }
    if (threadIdx.x <= a.b.drafts) {
        const uint32_t i = threadIdx.x;
        a.tokens[(uint64_t)seq * (a.b.drafts + 1) + i] = i < r ? a.b.tokens[(uint64_t)seq * a.b.drafts + i] : i == r ? pick : (uint32_t)LV_NO_TOKEN;
    }
}

// grid (seqs).  `accepted` is what the sums' launch found
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a)
{
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63;
    const uint32_t r = a.accepted[seq], count = a.b.counts ? min(a.b.counts[seq], a.b.drafts) : a.b.drafts;
    const bool mine = lane < a.segments;      // 64 at most
    const double rest = mine ? a.sums[((uint64_t)seq * a.segments + lane) * 2] : 0.0, whole = mine ? a.sums[((uint64_t)seq * a.segments + lane) * 2 + 1] : 0.0;
    verify_pick(a, seq, r, verify_row(a.b, seq, r, count), rest, whole);
}

// Both at once, a segment for each of 16 waves.  Bound by a chain of loads (drafts, their probabilities, rows, the segment again), then by a compute unit's vector work
// in double: 8 us a call of one sequence of 8192 entries, 9.8 of 32000, 26 of 128256.  grid (seqs)
__global__ __launch_bounds__(1024) void verify_whole_kernel(VerifyArgs a)
{
    __shared__ double sums[16][2];
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t count;
    const uint32_t r = verify_standing(a.b, seq, count);
    const VerifyRow row = verify_row(a.b, seq, r, count);
    double rest = 0.0, whole = 0.0;
    verify_sums<4>(row, wave * a.length + 4 * lane, min((wave + 1) * a.length, a.b.vocab), 256, rest, whole);
    if (lane == 0) {
        sums[wave][0] = rest;
        sums[wave][1] = whole;
    }
    __syncthreads();
    const bool mine = lane < a.segments;
    rest = mine ? sums[lane][0] : 0.0;
    whole = mine ? sums[lane][1] : 0.0;
    if (threadIdx.x == 0) a.accepted[seq] = r;
    verify_pick(a, seq, r, row, rest, whole);
}

}  // namespace lv
