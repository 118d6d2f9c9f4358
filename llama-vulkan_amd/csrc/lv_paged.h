// lv_paged.h — attention of new tokens over the pages of their sequences (lv_kernel_paged_attention).
//
// A row is a new token and one of the heads that share a key head; scores are computed transposed, S^T = K Q^T, on
// v_mfma_f32_16x16x32: a lane then holds scores of ONE row (column lane % 16), so maximum, rescaling and sum are per-lane numbers, and the registers of
// S^T are the second operand of O^T = V^T P^T as they are (any order of the 32 keys of a product does, as long as both operands have the same).  V^T comes
// from row-major values through ds_read_b64_tr_b16, which hands lane i of 16 the column i of 4 rows.
//
// Scores are in units of log2, 2^12 on top of the weights of fp16 products (a weight below 2^-14 of the largest would be an fp16 subnormal), which the sum has
// as well.  Masked scores are -inf, the running maximum starts at kNothing, finite and below all scores: a row that sees nothing ends with a sum of 0 and is written as 0.
#pragma once

#include <type_traits>

#include "lv_common.h"
#include "lv_device.h"
#include "lv_paged_plan.h"

namespace lv {

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));      // where uint4, a class, would be kept in memory
typedef uint32_t pg_u2 __attribute__((ext_vector_type(2)));
typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef short pg_s8 __attribute__((ext_vector_type(8)));

enum { kPgF16 = 0, kPgBf16 = 1, kPgQ8 = 2, kPgQ4 = 3 };

struct PagedAttnArgs {
    PagedView c;
    PagedDeal deal;
    const uint32_t *starts, *lens, *table;
    uint32_t table_ld;
    const void *q;
    void *out;
    uint32_t ldq, ldo, type;
    float scale;                // times log2 e
    const float *sinks;
    uint32_t items;             // of a key head at most: what `part` has room for
    uint32_t round;             // items of a key head that the device's compute units take at once, or 0
    float *part, *part_ml;      // of cut items: [item][kv head][tile][dim], [item][kv head][tile][2]
};

// paged_page of a position that is the same in all lanes: as constant memory the table is read by scalar loads, which wait for nothing but themselves.  A vector
// load's wait is one for all loads before it: keys and values on their way.
__device__ __forceinline__ uint32_t paged_page_uniform(const PagedAttnArgs &a, const uint32_t *row, uint32_t position)
{
    const uint32_t at = __builtin_amdgcn_readfirstlane(position), i = at >> a.c.shift;
    uint32_t p = kNoPage;
    if (i < a.table_ld) p = *((const __attribute__((address_space(4))) uint32_t *)(uintptr_t)(row + i));
    return p < a.c.pages ? p : kNoPage;
}

constexpr float kNothing = -3e38f;      // a running maximum before the first score

// ---- which item ------------------------------------------------------------------------------------------------------------------
struct PagedItem {
    PagedSeq s;
    uint32_t seq, tile, part, parts, run;
    uint32_t first;                           // item of this tile's part 0
    bool any;
};

__device__ __forceinline__ uint32_t wave_running_sum_u32(uint32_t v)
{
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);      // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

__device__ __forceinline__ PagedSeq paged_seq_of(const PagedAttnArgs &a, uint32_t b)
{
    return paged_seq(a.starts[b], a.starts[b + 1], a.lens[b], a.deal.tokens, a.deal.positions);
}

struct PagedLook {
    PagedSeq s;
    uint32_t tiles, steps;
};
__device__ __forceinline__ PagedLook paged_look(const PagedAttnArgs &a, uint32_t b)
{
    PagedLook x{};
    x.steps = 1;
    if (b < a.deal.seqs) {
        x.s = paged_seq_of(a, b);
        x.tiles = paged_tiles(a.deal, x.s);
        x.steps = paged_steps(a.deal, x.s);
    }
    return x;
}

// The sequence that an item (BY_ROW false) or a row of the tensors (true; `sub`: which of the heads that share a key head) belongs to, found by each wave on its own.  The run
// follows from the steps of all tiles of all sequences, summed up in the same order by every wave of both launches.  (1024 sequences of one token behind 63, 8 key heads: 157 us with
// lengths and steps looked at where nothing is cut, 131 without.)
template <bool BY_ROW> __device__ __forceinline__ PagedItem paged_locate(const PagedAttnArgs &a, uint32_t which, int lane, uint32_t sub = 0)
{
    PagedItem it{};
    uint32_t before = 0;
    auto found = [&](uint32_t b0, const PagedLook &x) {
        const uint32_t parts = paged_parts(x.steps, it.run), upto = before + wave_running_sum_u32(x.tiles * parts);
        const uint64_t here = __ballot(BY_ROW ? which >= x.s.row0 && which - x.s.row0 < x.s.rows : upto > which);
        if (!here) {
            before = __builtin_amdgcn_readlane(upto, 63);
            return false;
        }
        const int l = __builtin_ctzll(here);
        const uint32_t n = __builtin_amdgcn_readlane(x.tiles, l);
        it.seq = b0 + l;
        it.parts = __builtin_amdgcn_readlane(parts, l);
        it.s.row0 = __builtin_amdgcn_readlane(x.s.row0, l);
        it.s.rows = __builtin_amdgcn_readlane(x.s.rows, l);
        it.s.pos0 = (int32_t)__builtin_amdgcn_readlane((uint32_t)x.s.pos0, l);
        it.s.keys = __builtin_amdgcn_readlane(x.s.keys, l);
        it.any = true;
        const uint32_t start = __builtin_amdgcn_readlane(upto, l) - n * it.parts;
        // tiles that see most go first
        const uint32_t back = BY_ROW ? n - 1 - ((which - it.s.row0) * a.deal.group + sub) / a.deal.tile : (which - start) / it.parts;
        it.tile = n - 1 - back;
        it.first = start + back * it.parts;
        it.part = BY_ROW ? 0 : which - it.first;
        return true;
    };
    if (a.deal.seqs <= 64) {
        const PagedLook x = paged_look(a, lane);
        it.run = __builtin_amdgcn_readfirstlane(paged_run(a.deal, a.deal.target ? wave_sum((float)x.tiles * (float)x.steps) : 0.f));
        (void)found(0, x);
        return it;
    }
    if (BY_ROW || a.deal.target) {
        float all = 0.f;
        for (uint32_t b0 = 0; b0 < a.deal.seqs; b0 += 64) {
            const PagedLook x = paged_look(a, b0 + lane);
            all += wave_sum((float)x.tiles * (float)x.steps);
        }
        it.run = __builtin_amdgcn_readfirstlane(paged_run(a.deal, all));
        for (uint32_t b0 = 0; b0 < a.deal.seqs; b0 += 64)
            if (found(b0, paged_look(a, b0 + lane))) return it;
        return it;
    }
    // nothing is cut: the tiles follow from the rows alone, 256 sequences at a time
    it.run = paged_run(a.deal, 0.f);
    constexpr uint32_t W = 4;
    for (uint32_t b0 = 0; b0 < a.deal.seqs; b0 += 64 * W) {
        uint32_t from[W], to[W];
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
            const uint32_t b = min(b0 + 64 * w + lane, a.deal.seqs - 1);
            from[w] = a.starts[b];
            to[w] = a.starts[b + 1];
        }
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
            const bool is = b0 + 64 * w + lane < a.deal.seqs;
            PagedSeq s{};
            s.rows = is && min(to[w], a.deal.tokens) > from[w] ? min(to[w], a.deal.tokens) - from[w] : 0;
            const uint32_t tiles = paged_tiles(a.deal, s), upto = before + wave_running_sum_u32(tiles);
            const uint64_t here = __ballot(upto > which);
            if (here) {
                const int l = __builtin_ctzll(here);
                const uint32_t n = __builtin_amdgcn_readlane(tiles, l);
                it.seq = b0 + 64 * w + l;
                const PagedSeq found_s = paged_seq_of(a, it.seq);
                it.s.row0 = __builtin_amdgcn_readfirstlane(found_s.row0);
                it.s.rows = __builtin_amdgcn_readfirstlane(found_s.rows);
                it.s.pos0 = (int32_t)__builtin_amdgcn_readfirstlane((uint32_t)found_s.pos0);
                it.s.keys = __builtin_amdgcn_readfirstlane(found_s.keys);
                it.parts = 1;
                it.any = true;
                it.tile = n - 1 - (which - (__builtin_amdgcn_readlane(upto, l) - n));
                it.first = which;
                return it;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    return it;
}

// ---- elements ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float pg_exp2(float x) { return __builtin_amdgcn_exp2f(x); }      // 1 ulp; 0 below 2^-126

// eight 16-bit numbers of one kind
template <bool BF> __device__ __forceinline__ void pg_unpack8(uint4 u, float (&x)[8])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = BF ? __uint_as_float(w[i] << 16) : half_bits_to_float((uint16_t)w[i]);
        x[2 * i + 1] = BF ? __uint_as_float(w[i] & 0xffff0000u) : half_bits_to_float((uint16_t)(w[i] >> 16));
    }
}
__device__ __forceinline__ uint32_t pg_bits(float x, bool half) { return half ? (uint32_t)float_to_half_bits(x) : (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x); }
template <bool BF> __device__ __forceinline__ uint4 pg_pack8(const float (&x)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = pg_bits(x[2 * i], !BF) | (pg_bits(x[2 * i + 1], !BF) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// eight elements of `type` from `at` on
__device__ __forceinline__ void pg_load8(const void *p, uint32_t type, uint64_t at, float (&x)[8])
{
    if (type == LV_F32) {
        const float4 *f = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        const float4 u = f[0], v = f[1];
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
        return;
    }
    const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
    if (type == LV_F16) pg_unpack8<false>(u, x);
    else pg_unpack8<true>(u, x);
}
__device__ __forceinline__ void pg_store8(void *p, uint32_t type, uint64_t at, const float (&x)[8])
{
    if (type == LV_F32) {
        float4 *f = reinterpret_cast<float4 *>(static_cast<float *>(p) + at);
        f[0] = make_float4(x[0], x[1], x[2], x[3]);
        f[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) = type == LV_F16 ? pg_pack8<false>(x) : pg_pack8<true>(x);
}
// N times eight elements, eight of them every `step`: asked for, and made numbers of later
template <int N> struct PgRow {
    pg_u4 u[N], v[N];
};
// WIDE: may they have 32 bits?
template <bool WIDE, int N> __device__ __forceinline__ void pg_ask_row(const void *p, uint32_t type, uint64_t at, uint32_t step, PgRow<N> &r)
{
    const uint32_t size = WIDE && type == LV_F32 ? 4 : 2;
    const uint8_t *f = static_cast<const uint8_t *>(p) + at * size;
#pragma unroll
    for (int n = 0; n < N; n++) {
        r.u[n] = *reinterpret_cast<const pg_u4 *>(f + n * step * size);
        if constexpr (WIDE) r.v[n] = *reinterpret_cast<const pg_u4 *>(f + n * step * size + (size == 4 ? 16 : 0));
    }
}
template <bool WIDE, int N> __device__ __forceinline__ void pg_row_numbers(uint32_t type, const PgRow<N> &r, float (&x)[N][8])
{
    if (WIDE && type == LV_F32) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            #pragma unroll
            for (int e = 0; e < 8; e++) x[n][e] = __uint_as_float(e < 4 ? r.u[n][e % 4] : r.v[n][e % 4]);
        }
    } else if (type == LV_F16) {
#pragma unroll
        for (int n = 0; n < N; n++) pg_unpack8<false>(__builtin_bit_cast(uint4, r.u[n]), x[n]);
    } else {
#pragma unroll
        for (int n = 0; n < N; n++) pg_unpack8<true>(__builtin_bit_cast(uint4, r.u[n]), x[n]);
    }
}

// codes to fp16: the byte under 0x64 is 1024 + byte
__device__ __forceinline__ uint32_t pg_pk_add(uint32_t a, float b)
{
    const pg_h2 r = __builtin_bit_cast(pg_h2, a) + pg_h2{(_Float16)b, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t pg_pk_mul(uint32_t a, pg_h2 d) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(pg_h2, a) * d); }
// four bytes 0 .. 255 minus `bias`, as four fp16
__device__ __forceinline__ void pg_bytes_to_half(uint32_t w, float bias, uint32_t &lo, uint32_t &hi)
{
    lo = pg_pk_add(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), -1024.f - bias);
    hi = pg_pk_add(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u), -1024.f - bias);
}

template <bool BF> struct PgFrag { typedef pg_h8 type; };
template <> struct PgFrag<true> { typedef pg_b8 type; };
template <bool BF> __device__ __forceinline__ pg_f4 pg_mfma(typename PgFrag<BF>::type a, typename PgFrag<BF>::type b, pg_f4 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// x as a sum of N numbers of 16 bits: fp16 11 bits each, bf16 8
template <bool BF, int N, class Frag> __device__ __forceinline__ void pg_cut(float x, int e, Frag (&f)[N])
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        if constexpr (BF) {
            const __bf16 h = (__bf16)x;
            f[n][e] = h;
            x -= (float)h;
        } else {
            const _Float16 h = (_Float16)x;
            f[n][e] = h;
            x -= (float)h;
        }
    }
}

// s * f, rounded, less m
constexpr float kFar = 1048576.f;
__device__ __forceinline__ float pg_apart(float s, float f, float m)
{
#pragma clang fp contract(off)
    const float x = s * f;
    return x - m;
}

// what a result x is weighed with: w, but 1 where x is not finite and w has underflowed, 0 times which would be NaN
__device__ __forceinline__ float pg_weight(float x, float w) { return w == 0.f && x - x != 0.f ? 1.f : w; }

// bits where one of two 16-bit numbers is not finite
template <bool BF> __device__ __forceinline__ uint32_t pg_special(uint32_t w)
{
    return BF ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
// kind 0: the finite ones of eight numbers, 0 in place of others; 1, 2, 3: a one in place of each NaN, inf, -inf, 0 of others
template <bool BF> __device__ __forceinline__ typename PgFrag<BF>::type pg_only(typename PgFrag<BF>::type f, int kind)
{
    pg_s8 s = __builtin_bit_cast(pg_s8, f);
    constexpr int EX = BF ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int h = (uint16_t)s[e], size = h & 0x7fff;
        const bool finite = size < EX, yes = kind == 1 ? size > EX : h == (kind == 2 ? EX : EX | 0x8000);
        s[e] = (short)(kind == 0 ? (finite ? h : 0) : yes ? (BF ? 0x3f80 : 0x3c00) : 0);
    }
    return __builtin_bit_cast(typename PgFrag<BF>::type, s);
}

// the columns of a 4 x 16 tile of 16-bit elements; each of 16 lanes names the 8 bytes at row lane / 4, columns 4 (lane % 4) ..
__device__ __forceinline__ pg_s4 pg_read_columns(const uint8_t *p)
{
    typedef __attribute__((address_space(3))) pg_s4 lds_s4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
}

// ---- rows: single tokens, drafts, 32-bit queries -----------------------------------------------------------------------------------
// A workgroup's tile is 16 QT rows; its four waves take turns of 32 keys and never wait for one another before the end, where their results are put
// together.  Keys of 16 bits go from memory to registers as the first operand, values, and codes and scales of both, through the wave's own 32 rows of LDS; the next
// turn's are asked for before this turn's are used.  Bound by the bytes of the cache where there are many (131072 keys of 8 heads in fp16 99 us, 5.4 TB/s; 64 sequences of 8 bits
// 174 us, 4.9 TB/s); with few keys by a chain of loads, each about 2000 clocks: lengths, the first pages, the first keys.
//
// NQ: pieces of a query, 1, or with 32-bit queries 2 (fp16 rows: 22 bits) or 3 (bf16 rows: 24 bits); the weights have as many, 2 of bf16 at least.  Rows of
// codes: keys enter as exact integers, a block's sum is scaled in fp32.  Values are scaled in fp16 (a rounding of 2^-11 of each, beside the 16-bit result's own); with
// 32-bit queries they enter as two fp16 pieces, which hold them exactly: 19 bits at most, the last of them 2^-24 or more, as the scale's is.
// FINE: rows of codes and an fp16 result.  Its own rounding is no coarser than the weights' and the scaled values' are, and with both the error is 1.6 times the result's
// rounding alone; the weights enter as two pieces, and it is 1.4 times (single tokens and drafts: 1 to 7 % of the time).  Beside a bf16 result neither shows.
template <int BYTES> struct PgWord { typedef uint32_t type; };
template <> struct PgWord<8> { typedef pg_u2 type; };
// waves a SIMD that the registers are cut for: as many as leave none in memory, but two where 32 rows of 32-bit queries over fp16 rows (27 registers in memory) or rows of
// 8 bits (17) have heads of 128
constexpr int paged_rows_waves(int D, int CT, int NQ, int QT)
{
    if (D == 256) return 1;
    if (D == 128 && QT == 2 && NQ == 3) return 1;      // here 59 registers in memory cost more than a second wave gains (1024 tokens, the last of 4096: 340 us and 281)
    if (D == 128) return QT == 1 && NQ == 1 && CT >= kPgQ8 ? 3 : 2;
    return NQ > 1 && QT == 2 ? 2 : 3;
}

template <int D, int CT, int NQ, int QT, bool FINE>
__global__ __launch_bounds__(256, paged_rows_waves(D, CT, NQ, QT)) void paged_rows_kernel(PagedAttnArgs a)
{
    constexpr bool BF = CT == kPgBf16, BLOCKS = CT == kPgQ8 || CT == kPgQ4, EXACT = NQ > 1;
    constexpr int KS = D / 32, DT = D / 16, CH = D / 8, ROW = 2 * D + 16, NP = (BF || FINE) && NQ == 1 ? 2 : NQ, TILE = 16 * QT;
    constexpr float kLift = BF ? 0.f : 12.f, kRoom = 3.f;
    constexpr int MERGE = D + 4;                      // floats of a row of results in LDS
    typedef typename PgFrag<BF>::type Frag;
    constexpr int PLANES = BLOCKS && EXACT ? 2 : 1, VALUES = 32 * ROW * PLANES;      // bytes of a wave's 32 rows of values; 16 more a row put the 16 rows of a column read on all banks evenly
    __shared__ __attribute__((aligned(128))) uint8_t lds[4 * VALUES > 4 * 16 * MERGE * 4 ? 4 * VALUES : 4 * 16 * MERGE * 4];      // at the end 16 rows of results of each wave
    __shared__ float ml[4][TILE][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    const uint32_t head = blockIdx.x % a.c.kv_heads, item = blockIdx.x / a.c.kv_heads;
    const PagedItem it = paged_locate<false>(a, item, lane);
    if (!it.any) return;
    const uint32_t group = a.deal.group, rows = it.s.rows * group, r0 = it.tile * TILE;
    const uint32_t psize = 1u << a.c.shift;

    // this lane's rows: asked for here, made operands of when the first keys and values are on their way too
    constexpr int QS = CT == kPgQ4 ? 2 * KS : KS;
    PgRow<QS> raw[QT];
    uint32_t lo[QT], span[QT];      // the keys it sees: lo .. lo + span - 1
#pragma unroll
    for (int i = 0; i < QT; i++) {
        const uint32_t r = r0 + i * 16 + l16;
        const bool is = r < rows;
        const uint32_t tk = is ? r / group : 0, h = head * group + (is ? r - tk * group : 0);
        const int32_t p = it.s.pos0 + (int32_t)tk;
        lo[i] = p >= 0 ? paged_first_key((uint32_t)p, a.deal.window, a.deal.chunk) : 0;
        const uint32_t end = p >= 0 ? min((uint32_t)p + 1, it.s.keys) : 0;
        span[i] = is && end > lo[i] ? end - lo[i] : 0;
        const uint64_t at = (uint64_t)(it.s.row0 + tk) * a.ldq + (uint64_t)h * D;
        if constexpr (CT == kPgQ4) pg_ask_row<EXACT, QS>(a.q, a.type, at + (g4 / 2) * 8, 16, raw[i]);
        else pg_ask_row<EXACT, QS>(a.q, a.type, at + g4 * 8, 32, raw[i]);
    }
    // keys that any row sees, and those that all rows see
    const uint32_t last_row = min(r0 + TILE, rows) - 1;
    const int32_t p_first = it.s.pos0 + (int32_t)(r0 / group), p_last = it.s.pos0 + (int32_t)(last_row / group);
    const uint32_t k_lo = p_first >= 0 ? paged_first_key((uint32_t)p_first, a.deal.window, a.deal.chunk) : 0;
    const uint32_t k_hi = p_last >= 0 ? min((uint32_t)p_last + 1, it.s.keys) : 0;
    const uint32_t all_lo = p_last >= 0 ? paged_first_key((uint32_t)p_last, a.deal.window, a.deal.chunk) : 0, all_hi = p_first >= 0 ? (uint32_t)p_first + 1 : 0;
    const uint32_t base = k_lo & ~31u, n_steps = k_hi > base ? (k_hi - base + kPagedStep - 1) / kPagedStep : 0;
    const uint32_t s0 = paged_cut(n_steps, it.part, it.parts), s1 = paged_cut(n_steps, it.part + 1, it.parts);

    const uint32_t *table = a.table + (uint64_t)it.seq * a.table_ld;
    const uint32_t turns = n_steps ? (k_hi - base + 31) / 32 : 0, t_end = min(s1 * 4, turns);
    uint8_t *mine = lds + wave * VALUES;

    // row of 32 and unit of 16 bytes of the row that this lane brings with its i-th load of values, and of keys that are codes
    constexpr int UNITS = BLOCKS ? (CT == kPgQ8 ? D : D / 2) / 16 : CH, LOADS = UNITS > 1 ? 32 * UNITS / 64 : 1;
    // the scales of 32 rows are asked for as words in one load
    constexpr int WORD = D == 256 ? 8 : 4, WORDS = 2 * D / WORD;
    typedef typename PgWord<WORD>::type Word;
    struct Turn {
        pg_u4 k4[BLOCKS ? 1 : 2][BLOCKS ? LOADS : KS], v4[LOADS];
        Word ks, vs;
    };
    // (addresses are made anew in every turn, from a lane number that the compiler cannot see through: kept, they would take a hundred registers)
    int ln = lane;
    auto row_of = [&](int i) { return UNITS > 1 ? (i * 64 + ln) / UNITS : ln % 32; };
    auto unit_of = [&](int i) { return (i * 64 + ln) % UNITS; };
    // where 16 keys' codes lie (of keys; of values and scales at the same distances in every block), null without a page
    Turn x;
    auto place = [&](uint32_t t, int kt, uint32_t &in) {
        const uint32_t at = base + t * 32 + 16 * kt, page = paged_page_uniform(a, table, at);
        in = at & (psize - 1);
        return page;
    };
    auto block_of = [&](uint32_t page) { return a.c.data + ((uint64_t)(page != kNoPage ? page : 0) * a.c.kv_heads + head) * a.c.block; };
    const uint32_t scales_at = a.c.code_row << a.c.shift;
    auto load_keys = [&](uint32_t page0, uint32_t page1, uint32_t in0, uint32_t in1) {
        if constexpr (BLOCKS) {
            const uint8_t *block0 = block_of(page0), *block1 = block_of(page1);
            const uint8_t *pk0 = block0 + in0 * a.c.code_row, *pk1 = block1 + in1 * a.c.code_row;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int row = row_of(i), u = unit_of(i);
                const bool second = 64 / UNITS <= 16 ? i * (64 / UNITS) >= 16 : row >= 16;
                x.k4[0][i] = *reinterpret_cast<const pg_u4 *>((second ? pk1 : pk0) + (uint32_t)((row & 15) * (UNITS * 16) + u * 16));
            }
            const uint32_t at = (uint32_t)(ln % WORDS) * WORD;
            const uint8_t *ps = (at < D ? block0 + in0 * a.c.scale_row : block1 + in1 * a.c.scale_row) + scales_at + at % D;
            x.ks = *reinterpret_cast<const Word *>(ps);
            x.vs = *reinterpret_cast<const Word *>(ps + a.c.half);
        } else {
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const uint8_t *pk = block_of(kt ? page1 : page0) + (kt ? in1 : in0) * a.c.code_row;
#pragma unroll
                for (int k = 0; k < KS; k++) x.k4[kt][k] = *reinterpret_cast<const pg_u4 *>(pk + (uint32_t)((ln & 15) * (2 * D) + k * 64 + (ln >> 4) * 16));
            }
        }
    };
    auto load_values = [&](uint32_t page0, uint32_t page1, uint32_t in0, uint32_t in1) {
        const uint8_t *pv0 = block_of(page0) + a.c.half + in0 * a.c.code_row, *pv1 = block_of(page1) + a.c.half + in1 * a.c.code_row;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int row = row_of(i), u = unit_of(i);
            const bool second = 64 / UNITS <= 16 ? i * (64 / UNITS) >= 16 : row >= 16;      // of 16 keys; where a load covers no more, the same in all lanes
            x.v4[i] = *reinterpret_cast<const pg_u4 *>((second ? pv1 : pv0) + (uint32_t)((row & 15) * (UNITS * 16) + u * 16));
        }
    };
    // Codes of keys, and scales, pass through the place of the values, which is free then: loads of 16 bytes in a row and one for 32 rows' scales, where each lane's own
    // 4 or 8 bytes of a row would take three times the loads and four times the caches' accesses.  Units of a row change places by its number, so that 64 lanes read all banks.
    constexpr int KSC = 32 * UNITS * 16, VSC = KSC + 2 * D;
    auto unit_at = [&](int row, int u) { return row * (UNITS * 16) + (u ^ (row * UNITS / 16 & (UNITS - 1))) * 16; };
    pg_u2 kw[BLOCKS ? 2 : 1][BLOCKS ? KS : 1];      // codes of key (lane & 15)
    pg_u2 ks[BLOCKS ? 2 : 1][BLOCKS ? KS : 1];                              // scales of keys 4 g .. 4 g + 3 of 16: [key][block]
    uint16_t vd[BLOCKS ? LOADS : 1];
    auto turn_keys = [&]() {
#pragma unroll
        for (int i = 0; i < LOADS; i++) *reinterpret_cast<pg_u4 *>(mine + unit_at(row_of(i), unit_of(i))) = x.k4[0][i];
        const int at = ln % WORDS * WORD;
        *reinterpret_cast<Word *>(mine + KSC + at) = x.ks;
        *reinterpret_cast<Word *>(mine + VSC + at) = x.vs;
    };
    auto take_keys = [&]() {
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int row = kt * 16 + (ln & 15), g = ln >> 4;
                if constexpr (CT == kPgQ8) {
                    kw[kt][k] = *reinterpret_cast<const pg_u2 *>(mine + unit_at(row, 2 * k + g / 2) + g % 2 * 8);
                } else {
                    kw[kt][k].x = *reinterpret_cast<const uint32_t *>(mine + unit_at(row, k) + g * 4);
                }
                ks[kt][k] = *reinterpret_cast<const pg_u2 *>(mine + KSC + (kt * 16 + g * 4) * (D / 16) + k * 8);
            }
#pragma unroll
        for (int i = 0; i < LOADS; i++) vd[i] = *reinterpret_cast<const uint16_t *>(mine + VSC + row_of(i) * (D / 16) + (CT == kPgQ8 ? unit_of(i) / 2 : unit_of(i)) * 2);
    };

    pg_f4 o[DT][QT];
    float m[QT], l[QT];
#pragma unroll
    for (int i = 0; i < QT; i++) {
        m[i] = kNothing;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d][i] = pg_f4{0.f, 0.f, 0.f, 0.f};
    }
    // eight elements into chunk `ch` of a row of values in LDS
    auto put = [&](int row, int ch, uint4 w, int plane = 0) { *reinterpret_cast<uint4 *>(mine + plane * (32 * ROW) + row * ROW + ch * 16) = w; };
    // first operand of O^T for dimensions 16 d ..: dimension (ln & 15), keys 4 g .. + 3 and 16 + 4 g .. + 3
    auto values = [&](int d, int plane = 0) {
        const uint8_t *at = mine + (4 * (ln >> 4) + (ln & 15) / 4) * ROW + 8 * (ln & 3) + 32 * d + plane * (32 * ROW);
        const pg_s4 u = pg_read_columns(at), v = pg_read_columns(at + 16 * ROW);
        return __builtin_bit_cast(Frag, pg_s8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
    };

    // does row i see key 16 kt + 4 g + r of a turn?
    auto sees = [&](uint32_t kb, bool ok, int i, int kt, int r) { return kb + (kt * 16 + (ln >> 4) * 4 + r) - lo[i] < (ok ? span[i] : 0u); };
    // Values that no row sees are made 0: a page's rows behind the sequence's end may hold anything, and 0 times that has to be 0.
    auto clear = [&](uint32_t kb, bool ok0, bool ok1) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int row = row_of(i);
            const bool keep = kb + row - k_lo < ((row < 16 ? ok0 : ok1) ? k_hi - k_lo : 0u);
            if constexpr (CT <= kPgBf16) {
                if (!keep) x.v4[i] = pg_u4{0, 0, 0, 0};
            } else {
                if (!keep) vd[i] = 0;
            }
        }
    };
    auto any_special = [&]() {
        uint32_t odd = 0;
        if constexpr (CT <= kPgBf16) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) odd |= pg_special<BF>(x.v4[i].x) | pg_special<BF>(x.v4[i].y) | pg_special<BF>(x.v4[i].z) | pg_special<BF>(x.v4[i].w);
        }
        return __any(odd != 0);
    };
    bool special = false;
    const uint32_t t_first = s0 * 4 + wave;
    uint32_t t = t_first, page0 = kNoPage, page1 = kNoPage, in0 = 0, in1 = 0, next0 = kNoPage, next1 = kNoPage;
    if (t < t_end) {
        page0 = place(t, 0, in0);
        page1 = place(t, 1, in1);
        load_keys(page0, page1, in0, in1);
        load_values(page0, page1, in0, in1);
        // (the last turn asks for its own again, which are in the caches: a condition around the loads costs registers)
        if constexpr (BLOCKS) {
            const uint32_t next = t + 4 < t_end ? t + 4 : t;
            next0 = place(next, 0, in0);
            next1 = place(next, 1, in1);
        }
    }

    Frag q[QT][KS][NQ];
    float factor[QT];
#pragma unroll
    for (int i = 0; i < QT; i++) {
        float u[QS][8], z[KS][8], top = 0.f;
        pg_row_numbers<EXACT, QS>(a.type, raw[i], u);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if constexpr (CT == kPgQ4) {      // byte 4 g + j of a block holds elements 4 g + j and 16 + 4 g + j
                    const float a0 = u[2 * k + e / 4][e % 4], a1 = u[2 * k + e / 4][4 + e % 4];
                    z[k][e] = g4 & 1 ? a1 : a0;
                } else {
                    z[k][e] = u[k][e];
                }
                top = fmaxf(top, fabsf(z[k][e]));
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // a power of two brings the row's largest element to 2^10 .. 2^11: no overflow, and small pieces are no subnormals
        int e2 = (int)(__float_as_uint(top) >> 23) - 127 - 10;
        if (e2 > 117 || e2 < -110) e2 = 0;      // inf, NaN; 0 and numbers next to it
        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
        factor[i] = a.scale * __uint_as_float((uint32_t)(127 + e2) << 23);
        const bool is = r0 + i * 16 + l16 < rows;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) pg_cut<BF, NQ>(is ? z[k][e] * down : 0.f, e, q[i][k]);
    }

    for (; t < t_end; t += 4) {
        asm volatile("" : "+v"(ln));
        const uint32_t kb = base + t * 32;
        const bool ok0 = page0 != kNoPage, ok1 = page1 != kNoPage;
        const bool inside = kb >= k_lo && kb + 32 <= k_hi && ok0 && ok1;                // every key of the turn is some row's
        const bool edge = kb < all_lo || kb + 32 > all_hi || !inside;                   // some row does not see all of them
        // The next turn's keys are asked for as soon as this turn's are used up, its values likewise; their pages are known from the turn before
        const uint32_t next = t + 4 < t_end ? t + 4 : t;
        if constexpr (!BLOCKS) {
            next0 = place(next, 0, in0);
            next1 = place(next, 1, in1);
        }
        page0 = next0;
        page1 = next1;
        const uint32_t at0 = in0, at1 = in1;
        if constexpr (BLOCKS) {
            turn_keys();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            load_keys(page0, page1, at0, at1);
            take_keys();
        }
        if constexpr (BLOCKS) {
            const uint32_t then = next + 4 < t_end ? next + 4 : next;
            next0 = place(then, 0, in0);
            next1 = place(then, 1, in1);
        }
        pg_f4 sc[2][QT];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
#pragma unroll
            for (int i = 0; i < QT; i++) sc[kt][i] = pg_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                Frag f;
                if constexpr (CT <= kPgBf16) {
                    f = __builtin_bit_cast(Frag, x.k4[kt][k]);
                } else {
                    uint4 w;
                    if constexpr (CT == kPgQ8) {
                        pg_bytes_to_half(kw[kt][k].x ^ 0x80808080u, 128.f, w.x, w.y);
                        pg_bytes_to_half(kw[kt][k].y ^ 0x80808080u, 128.f, w.z, w.w);
                    } else {
                        pg_bytes_to_half(kw[kt][k].x & 0x0f0f0f0fu, 8.f, w.x, w.y);
                        pg_bytes_to_half((kw[kt][k].x >> 4) & 0x0f0f0f0fu, 8.f, w.z, w.w);
                    }
                    f = __builtin_bit_cast(Frag, w);
                }
#pragma unroll
                for (int i = 0; i < QT; i++) {
                    pg_f4 acc = BLOCKS ? pg_f4{0.f, 0.f, 0.f, 0.f} : sc[kt][i];
#pragma unroll
                    for (int n = NQ - 1; n >= 0; n--) acc = pg_mfma<BF>(f, q[i][k][n], acc);
                    if constexpr (BLOCKS) {
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int at = r * KS + k;      // half at / of ks: [key][block]
                            const uint32_t word = at % 4 < 2 ? ks[kt][at / 4].x : ks[kt][at / 4].y;
                            sc[kt][i][r] = fmaf(half_bits_to_float((uint16_t)(word >> (at % 2 * 16))), acc[r], sc[kt][i][r]);
                        }
                    } else {
                        sc[kt][i] = acc;
                    }
                }
            }
        }
        if constexpr (!BLOCKS) load_keys(page0, page1, at0, at1);
        Frag p[QT][NP];
#pragma unroll
        for (int i = 0; i < QT; i++) {
            float s[8], top = m[i];
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = sc[e / 4][i][e % 4] * factor[i];
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[e] = sees(kb, e < 4 ? ok0 : ok1, i, e / 4, e % 4) ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, s[e]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            // the reference follows the maximum where it is more than kRoom behind: weights stay below 2^15, and most turns leave the results as they are
            if (__any(top > m[i] + kRoom)) {
                const float f = pg_exp2(m[i] - top);
                m[i] = top;
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[d][i][r] *= f;
            }
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float w = pg_exp2(s[e] - m[i] + kLift);
                sum += w;
                pg_cut<BF, NP>(w, e, p[i]);
            }
            l[i] += sum;
        }
        if (!inside) clear(kb, ok0, ok1);
        // Numbers that are not finite are left out here and added apart, behind the loop, to the rows that see them: a weight that is 0, or a negative piece of
        // one, would spread them or turn their sign.
        if (CT <= kPgBf16 && any_special()) {
            special = true;
#pragma unroll
            for (int i = 0; i < (CT <= kPgBf16 ? LOADS : 0); i++) x.v4[i] = __builtin_bit_cast(pg_u4, pg_only<BF>(__builtin_bit_cast(Frag, x.v4[i]), 0));
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int row = row_of(i), u = unit_of(i);
            if constexpr (CT <= kPgBf16) {
                put(row, u, __builtin_bit_cast(uint4, x.v4[i]));
            } else {
                const pg_u4 c = x.v4[i];
                const _Float16 d = __builtin_bit_cast(_Float16, vd[i]);
                auto values_of = [&](uint32_t c0, uint32_t c1, float bias, int ch) {      // eight bytes' numbers into a chunk
                    uint4 w;
                    pg_bytes_to_half(c0, bias, w.x, w.y);
                    pg_bytes_to_half(c1, bias, w.z, w.w);
                    if constexpr (EXACT) {
                        const pg_h8 code = __builtin_bit_cast(pg_h8, w);
                        pg_h8 piece[2];
#pragma unroll
                        for (int e = 0; e < 8; e++) pg_cut<false, 2>((float)code[e] * (float)d, e, piece);
                        put(row, ch, __builtin_bit_cast(uint4, piece[0]));
                        put(row, ch, __builtin_bit_cast(uint4, piece[1]), 1);
                    } else {
                        const pg_h2 dd = {d, d};
                        put(row, ch, make_uint4(pg_pk_mul(w.x, dd), pg_pk_mul(w.y, dd), pg_pk_mul(w.z, dd), pg_pk_mul(w.w, dd)));
                    }
                };
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if constexpr (CT == kPgQ8) {
                        values_of(c[2 * j] ^ 0x80808080u, c[2 * j + 1] ^ 0x80808080u, 128.f, 2 * u + j);
                    } else {
                        values_of(c[2 * j] & 0x0f0f0f0fu, c[2 * j + 1] & 0x0f0f0f0fu, 8.f, 4 * u + j);
                        values_of((c[2 * j] >> 4) & 0x0f0f0f0fu, (c[2 * j + 1] >> 4) & 0x0f0f0f0fu, 8.f, 4 * u + 2 + j);
                    }
                }
            }
        }
        load_values(page0, page1, at0, at1);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if constexpr (PLANES == 2) {      // the smaller pieces first; the product of both smaller ones is 2^-22 of the whole
                const Frag v = values(d, 1);
#pragma unroll
                for (int i = 0; i < QT; i++) o[d][i] = pg_mfma<BF>(v, p[i][0], o[d][i]);
            }
            const Frag v = values(d);
#pragma unroll
            for (int i = 0; i < QT; i++)
#pragma unroll
                for (int n = NP - 1; n >= 0; n--) o[d][i] = pg_mfma<BF>(v, p[i][n], o[d][i]);
        }
    }

    if (CT <= kPgBf16 && special) {
        for (t = t_first; t < t_end; t += 4) {
            const uint32_t kb = base + t * 32;
            page0 = place(t, 0, in0);
            page1 = place(t, 1, in1);
            const bool ok0 = page0 != kNoPage, ok1 = page1 != kNoPage;
            load_values(page0, page1, in0, in1);
            clear(kb, ok0, ok1);
            if (!any_special()) continue;
#pragma unroll
            for (int i = 0; i < (CT <= kPgBf16 ? LOADS : 0); i++) put(row_of(i), unit_of(i), __builtin_bit_cast(uint4, x.v4[i]));
            // 1: NaN, 2: inf, 3: -inf.  Counts of each among the keys that a row sees, as a product of ones
#pragma unroll 1
            for (int kind = 1; kind <= 3; kind++) {
                const float add = kind == 1 ? __builtin_nanf("") : kind == 2 ? INFINITY : -INFINITY;
                Frag one[QT];
#pragma unroll
                for (int i = 0; i < QT; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float w = sees(kb, e < 4 ? ok0 : ok1, i, e / 4, e % 4) ? 1.f : 0.f;
                        if constexpr (BF) one[i][e] = (__bf16)w;
                        else one[i][e] = (_Float16)w;
                    }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const Frag v = pg_only<BF>(values(d), kind);
#pragma unroll
                    for (int i = 0; i < QT; i++) {
                        const pg_f4 n = pg_mfma<BF>(v, one[i], pg_f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int r = 0; r < 4; r++) o[d][i][r] += n[r] > 0.f ? add : 0.f;
                    }
                }
            }
        }
    }

    // the four waves' results put together, 16 rows at a time
#pragma unroll
    for (int i = 0; i < QT; i++) {
        float sum = l[i];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g4 == 0) {
            ml[wave][i * 16 + l16][0] = m[i];
            ml[wave][i * 16 + l16][1] = sum;
        }
    }
    float *res = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int i = 0; i < QT; i++) {
        __syncthreads();      // ml, and the values of all waves are read; then the 16 rows before these
        float top = ml[0][i * 16 + l16][0];
#pragma unroll
        for (int w = 1; w < 4; w++) top = fmaxf(top, ml[w][i * 16 + l16][0]);
        const float f = pg_exp2(m[i] - top);
#pragma unroll
        for (int d = 0; d < DT; d++)
            *reinterpret_cast<float4 *>(res + (wave * 16 + l16) * MERGE + d * 16 + g4 * 4) = make_float4(o[d][i][0] * f, o[d][i][1] * f, o[d][i][2] * f, o[d][i][3] * f);
        if (CT <= kPgBf16 && special) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) res[(wave * 16 + l16) * MERGE + d * 16 + g4 * 4 + r] = o[d][i][r] * pg_weight(o[d][i][r], f);
        }
        __syncthreads();
        for (int u = threadIdx.x; u < 16 * CH; u += 256) {
            const int row = u / CH, c = u % CH * 8;
            const uint32_t r = r0 + i * 16 + row;
            if (r >= rows) continue;
            float y[8], ms[4];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = 0.f;
            float big = kNothing, all = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                ms[w] = ml[w][i * 16 + row][0];
                big = fmaxf(big, ms[w]);
                const float4 *s = reinterpret_cast<const float4 *>(res + (w * 16 + row) * MERGE + c);
                y[0] += s[0].x; y[1] += s[0].y; y[2] += s[0].z; y[3] += s[0].w;
                y[4] += s[1].x; y[5] += s[1].y; y[6] += s[1].z; y[7] += s[1].w;
            }
#pragma unroll
            for (int w = 0; w < 4; w++) all = fmaf(ml[w][i * 16 + row][1], pg_exp2(ms[w] - big), all);
            if (it.parts > 1) {
                const uint64_t at = ((uint64_t)item * a.c.kv_heads + head) * TILE + i * 16 + row;
                pg_store8(a.part, LV_F32, at * D + c, y);
                if (c == 0) {
                    a.part_ml[2 * at] = big;
                    a.part_ml[2 * at + 1] = all;
                }
                continue;
            }
            const uint32_t t2 = r / group, h = head * group + (r - t2 * group);
            float f2 = 1.f;
            if (a.sinks) {
                const float sink = a.sinks[h] * 1.44269504088896341f, over = fmaxf(big, sink);
                f2 = pg_exp2(big - over);
                all = fmaf(all, f2, pg_exp2(sink - over + kLift));
            }
            f2 = all == 0.f ? 0.f : f2 / all;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = all == 0.f ? 0.f : y[e] * (CT <= kPgBf16 ? pg_weight(y[e], f2) : f2);
            pg_store8(a.out, a.type, (uint64_t)(it.s.row0 + t2) * a.ldo + (uint64_t)h * D + c, y);
        }
    }
}

// ---- tiles: chunks of a prompt -------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows of one key head, 32 a wave, and walks their keys in tiles of 64 that all four waves share, double-buffered in LDS by direct
// loads; two workgroups a CU, so that one's softmax fills the other's products.  v_mfma_f32_32x32x16: S^T = K Q^T leaves 32 scores of one row in a lane
// (and 32 in lane ^ 32), and eight registers in a row are an operand of O^T = V^T P^T whose other one comes through ds_read_b64_tr_b16.
// A wave reads 32 KB of LDS and issues 32 products of 32 clocks for a tile, its share of the LDS's rate and a SIMD's: bound by both, then by the softmax's vector work.
// 2048 tokens behind 6144, 32 heads over 8 of 128, bf16: 239 us, 1010 TFLOP/s, matrix units at work 51 % of the time, vector units 45.
// The running maximum is a reference: weights are formed with it at once, and only where their sum says that a score is far above it are the maximum taken, the results
// rescaled and the weights formed anew.  Most tiles do without the maximum's 48 vector instructions (half of them make numbers canonical).
// Weights enter the second product as one fp16 (2^-11) or bf16 (2^-8) number: beside a 16-bit result's own rounding, over all the keys of a row.
// FINE: as two fp16 pieces, as above (1024 tokens, the last of 4096, 8 bits: 119 and 154 us; 4 bits 118 and 149).  Rows of codes come through registers instead of direct loads,
// some of which are in memory with heads of 128: 3 with 8 bits, 16 and 8 with 8 and 4 bits and FINE.
typedef float pg_f16v __attribute__((ext_vector_type(16)));


template <bool BF> __device__ __forceinline__ pg_f16v pg_mfma32(typename PgFrag<BF>::type a, typename PgFrag<BF>::type b, pg_f16v c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void pg_lds;

// N runs of 64 x 16 bytes from base + 1024 i + each lane's offset to LDS, lane after lane from to + 1024 i on.  The compiler would let every read of LDS wait for all
// direct loads that it knows of, and so for the tile after the one that is read; the loop's own wait, for the tile it is about to read, is all that is needed.  (2048
// tokens behind 6144: 279 us with the builtin, 313 through registers, 261 so.)  No register is written, so what is in flight behind the compiler's back is LDS only, which
// nobody reads yet.
template <int N> __device__ __forceinline__ void pg_load_direct(uint32_t to, const uint8_t *base, const uint32_t (&at)[N])
{
    static_assert(N == 2 || N == 4, "runs");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024\n\t"
                     "global_load_lds_dwordx4 %3, %5 offset:2048\n\tglobal_load_lds_dwordx4 %4, %5 offset:0xc00"
                     : : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "s"(base) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024"
                     : : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(at[0]), "v"(at[1]), "s"(base) : "memory", "m0");
}

constexpr int kPagedTileRows = 128;
constexpr float paged_tile_lift(bool bf) { return bf ? 0.f : 6.f; }      // of the weight of a score at the reference, log2

template <int D, int CT, bool FINE>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedAttnArgs a)
{
    constexpr bool BF = CT == kPgBf16, BLOCKS = CT == kPgQ8 || CT == kPgQ4;
    constexpr int KS = D / 16, DT = D / 32, CH = D / 8, ROW = 2 * D, STAGE = 2 * 64 * ROW, KB = D / 32;
    constexpr float kLift = paged_tile_lift(BF), MOST = 32768.f;      // of a lane's weights in a tile: each fits fp16
    typedef typename PgFrag<BF>::type Frag;
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * STAGE];      // stage: 64 rows of keys, 64 of values
    __shared__ __attribute__((aligned(16))) uint16_t key_scales[BLOCKS ? 2 * KB * 64 : 1];      // of a stage: [block][key]
    __shared__ uint32_t special;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, hh = lane >> 5;
    const uint32_t head = blockIdx.x % a.c.kv_heads;
    uint32_t item = blockIdx.x / a.c.kv_heads;
    // Items come with those first that see most.  The second workgroup of a compute unit is one of the next round, taken backwards: the sums of two come out even
    // (64 tiles of 8 key heads, 512 workgroups at once: 256 to 253 us)
    if (a.round && item / a.round % 2 && (item / a.round + 1) * a.round <= gridDim.x / a.c.kv_heads) item = item / a.round * a.round + (a.round - 1 - item % a.round);
    const PagedItem it = paged_locate<false>(a, item, lane);
    if (!it.any) return;
    if (threadIdx.x == 0) special = 0;      // ordered by the loop's barriers, and the one behind it
    const uint32_t group = a.deal.group, rows = it.s.rows * group, r0 = it.tile * kPagedTileRows, psize = 1u << a.c.shift;

    // keys that rows first .. last see, any of them and all of them
    struct Range {
        uint32_t lo, hi, all_lo, all_hi;
    };
    auto range = [&](uint32_t first, uint32_t last) {
        const int32_t p0 = it.s.pos0 + (int32_t)(first / group), p1 = it.s.pos0 + (int32_t)(last / group);
        Range r;
        r.lo = p0 >= 0 ? paged_first_key((uint32_t)p0, a.deal.window, a.deal.chunk) : 0;
        r.hi = p1 >= 0 ? min((uint32_t)p1 + 1, it.s.keys) : 0;
        r.all_lo = p1 >= 0 ? paged_first_key((uint32_t)p1, a.deal.window, a.deal.chunk) : 0;
        r.all_hi = p0 >= 0 ? min((uint32_t)p0 + 1, it.s.keys) : 0;
        return r;
    };
    const Range all = range(r0, min(r0 + kPagedTileRows, rows) - 1);
    const uint32_t w0 = r0 + wave * 32;
    const bool idle = w0 >= rows;      // no row of this wave: it brings its share of the tiles
    const Range own = range(idle ? r0 : w0, min(w0 + 32, rows) - 1);
    const uint32_t base = all.lo & ~31u, n_steps = all.hi > base ? (all.hi - base + kPagedStep - 1) / kPagedStep : 0;
    const uint32_t s0 = paged_cut(n_steps, it.part, it.parts), s1 = paged_cut(n_steps, it.part + 1, it.parts);
    const uint32_t tiles = n_steps ? (all.hi - base + 63) / 64 : 0, t_end = min(s1 * (kPagedStep / 64), tiles);
    const uint32_t *table = a.table + (uint64_t)it.seq * a.table_ld;

    // a wave brings 16 keys and their values, which lie in one page.  Chunks of 16 bytes are stored at places that depend on their row: keys are read by 32 rows at
    // once (chunk ^ row % 16), values by 4 rows x 64 bytes (groups of four chunks ^ row % 4; of two rows in 256 bytes, ^ half the row)
    constexpr int PER = 64 / CH, LOADS = 16 / PER;      // rows a load, loads
    // what a lane brings by its load i, less 1024 i: places in the wave's 16 rows
    uint32_t key_at[LOADS], value_at[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int row = i * PER + lane / CH, ch = lane % CH;
        key_at[i] = (uint32_t)(lane / CH * ROW + (ch ^ (row % (CH < 16 ? CH : 16))) * 16);
        value_at[i] = (uint32_t)(lane / CH * ROW + (ch ^ (CH == 8 ? (row / 2 % 2) * 4 : (row % 4) * 4)) * 16);
    }
    auto issue = [&](int st, uint32_t page, uint32_t in) {
        const uint8_t *keys = a.c.data + ((uint64_t)(page != kNoPage ? page : 0) * a.c.kv_heads + head) * a.c.block + in * ROW;
        const uint32_t to = (uint32_t)(uintptr_t)(pg_lds *)(lds + st * STAGE + wave * (16 * ROW));
        pg_load_direct(to, keys, key_at);
        pg_load_direct(to + 64 * ROW, keys + a.c.half, value_at);
    };
    // Rows of blocks go through registers: asked for a tile ahead, and stored as fp16 when the tile before is used up.  A unit is 16 codes of 8 bits, or 8 bytes of 4 bits;
    // keys become integers, whose blocks' sums are scaled in fp32, values are scaled here (2^-11 of each, beside the 16-bit result's own rounding).
    constexpr int UNITS = D / 16, BLOADS = BLOCKS ? 16 * UNITS / 64 : 1;      // of a row; a lane's
    typedef typename std::conditional<CT == kPgQ4, pg_u2, pg_u4>::type Unit;
    Unit ku[BLOADS], vu[BLOADS];
    uint32_t vs[BLOADS];
    uint16_t ks[KB];
    auto fetch = [&](uint32_t page, uint32_t in) {
        const uint8_t *block = a.c.data + ((uint64_t)(page != kNoPage ? page : 0) * a.c.kv_heads + head) * a.c.block;
        const uint8_t *keys = block + in * a.c.code_row, *scales = block + (a.c.code_row << a.c.shift) + in * a.c.scale_row;
#pragma unroll
        for (int i = 0; i < BLOADS; i++) {
            const int u = i * 64 + lane;
            ku[i] = *reinterpret_cast<const Unit *>(keys + (uint32_t)(u * sizeof(Unit)));
            vu[i] = *reinterpret_cast<const Unit *>(keys + a.c.half + (uint32_t)(u * sizeof(Unit)));
            vs[i] = *reinterpret_cast<const uint16_t *>(scales + a.c.half + (uint32_t)(u / 2 * 2));
        }
#pragma unroll
        for (int k = 0; k < KB; k++) ks[k] = *reinterpret_cast<const uint16_t *>(scales + (uint32_t)((lane & 15) * (2 * KB) + 2 * k));
    };
    auto store = [&](int st, uint32_t kb, bool ok) {
        uint8_t *kd = lds + st * STAGE + wave * (16 * ROW), *vd = kd + 64 * ROW;
#pragma unroll
        for (int i = 0; i < BLOADS; i++) {
            const int u = i * 64 + lane, row = u / UNITS, in = u % UNITS;
            const int c0 = CT == kPgQ8 ? 2 * in : in / 2 * 4 + in % 2, c1 = CT == kPgQ8 ? c0 + 1 : c0 + 2;
            const int kx = row % (CH < 16 ? CH : 16), vx = CH == 8 ? (row / 2 % 2) * 4 : (row % 4) * 4;
            const uint32_t key = kb + wave * 16 + row;
            const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)(key - all.lo < (ok ? all.hi - all.lo : 0u) ? vs[i] : 0u));      // values that no row sees: 0
            const pg_h2 dd = {d, d};
            uint32_t w[8];
            auto unpack = [&](const Unit &x) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (CT == kPgQ8) pg_bytes_to_half(x[e] ^ 0x80808080u, 128.f, w[2 * e], w[2 * e + 1]);
                    else pg_bytes_to_half((e < 2 ? x[e] : x[e - 2] >> 4) & 0x0f0f0f0fu, 8.f, w[2 * e], w[2 * e + 1]);
                }
            };
            unpack(ku[i]);
            *reinterpret_cast<pg_u4 *>(kd + row * ROW + (c0 ^ kx) * 16) = pg_u4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<pg_u4 *>(kd + row * ROW + (c1 ^ kx) * 16) = pg_u4{w[4], w[5], w[6], w[7]};
            unpack(vu[i]);
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = pg_pk_mul(w[e], dd);
            *reinterpret_cast<pg_u4 *>(vd + row * ROW + (c0 ^ vx) * 16) = pg_u4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<pg_u4 *>(vd + row * ROW + (c1 ^ vx) * 16) = pg_u4{w[4], w[5], w[6], w[7]};
        }
        if (lane < 16) {
#pragma unroll
            for (int k = 0; k < KB; k++) key_scales[(st * KB + k) * 64 + wave * 16 + lane] = ks[k];
        }
    };
    auto page_of = [&](uint32_t at) { return paged_page_uniform(a, table, at); };
    uint32_t t = s0 * (kPagedStep / 64), mine = kNoPage, here = kNoPage;
    if (t < t_end) {
        here = page_of(base + t * 64 + wave * 16);
        if constexpr (BLOCKS) fetch(here, (base + t * 64 + wave * 16) & (psize - 1));
        else issue(0, here, (base + t * 64 + wave * 16) & (psize - 1));
    }
    if (t + 1 < t_end) mine = page_of(base + (t + 1) * 64 + wave * 16);

    // this lane's row
    Frag q[KS];
    float factor;
    uint32_t lo, span;
    {
        const uint32_t r = w0 + l32;
        const bool is = r < rows;
        const uint32_t tk = is ? r / group : 0, h = head * group + (is ? r - tk * group : 0);
        const int32_t p = it.s.pos0 + (int32_t)tk;
        lo = p >= 0 ? paged_first_key((uint32_t)p, a.deal.window, a.deal.chunk) : 0;
        const uint32_t end = p >= 0 ? min((uint32_t)p + 1, it.s.keys) : 0;
        span = is && end > lo ? end - lo : 0;
        float z[KS][8], top = 0.f;
        PgRow<KS> raw;
        pg_ask_row<false, KS>(a.q, a.type, (uint64_t)(it.s.row0 + tk) * a.ldq + (uint64_t)h * D + hh * 8, 16, raw);
        pg_row_numbers<false, KS>(a.type, raw, z);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(z[k][e]));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        int e2 = (int)(__float_as_uint(top) >> 23) - 127 - 10;      // as in the kernel for rows
        if (e2 > 117 || e2 < -110) e2 = 0;
        const float down = copysignf(__uint_as_float((uint32_t)(127 - e2) << 23), a.scale);
        factor = fmaxf(fabsf(a.scale) * __uint_as_float((uint32_t)(127 + e2) << 23), 1e-37f);      // above 0: -inf times it is -inf
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                Frag one[1];
                pg_cut<BF, 1>(is ? z[k][e] * down : 0.f, e, one);
                q[k][e] = one[0][e];
            }
    }

    pg_f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    float m = kNothing, l = 0.f, less = -kNothing;      // less: kLift - m, or what lets the weights overflow

    // Which of a tile's four runs of 16 keys have a page?  All of them, unless one of the item's pages is missing: looked up once.
    uint32_t missing = 0;
    {
        const uint32_t k0 = base + s0 * kPagedStep, k1 = min(base + s1 * kPagedStep, all.hi);
        for (uint32_t i = (k0 >> a.c.shift) + lane; k0 < k1 && i <= (k1 - 1) >> a.c.shift; i += 64) missing |= i >= a.table_ld || table[i] >= a.c.pages ? 1u : 0u;
        missing = __any(missing != 0);
    }
    auto pages_of = [&](uint32_t kb) {
        if (!missing) return 15u;
        uint32_t ok = 0;
        for (int g = 0; g < 4; g++) ok |= (page_of(kb + 16 * g) != kNoPage ? 1u : 0u) << g;
        return ok;
    };
    // does some row of the workgroup not see some key of a tile?
    auto partly = [&](uint32_t kb, uint32_t ok) { return kb < all.all_lo || kb + 64 > all.all_hi || ok != 15; };
    // In such a tile values that no row sees become 0 (0 times what earlier users of a page left there has to be 0), and so do numbers that are not finite.  In other
    // tiles all rows see those, and what they make of a result shows in it.  Behind the loop results are put right where any were found.
    auto clean = [&](uint8_t *vals, uint32_t kb, uint32_t ok) {
        uint32_t odd = 0;
        for (int c = threadIdx.x; c < 64 * CH; c += 256) {
            const uint32_t row = c / CH;
            pg_u4 *w = reinterpret_cast<pg_u4 *>(vals + c * 16), x = *w;
            if (kb + row - all.lo < ((ok >> (row / 16)) & 1 ? all.hi - all.lo : 0u)) {
                const uint32_t here = pg_special<BF>(x[0]) | pg_special<BF>(x[1]) | pg_special<BF>(x[2]) | pg_special<BF>(x[3]);
                if (here) *w = __builtin_bit_cast(pg_u4, pg_only<BF>(__builtin_bit_cast(Frag, x), 0));
                odd |= here;
            } else {
                *w = pg_u4{0, 0, 0, 0};
            }
        }
        if (odd) special = 1;
        __syncthreads();
    };
    // values of 16 keys as the first operand for 32 dimensions: a lane has dimension l32, keys 4 hh .. + 3 and 8 + 4 hh .. + 3
    const int vrow = 4 * hh + (lane & 15) / 4, vx = CH == 8 ? (vrow / 2 % 2) * 4 : (vrow % 4) * 4, vch = (l32 / 16) * 2 + (lane & 3) / 2, voff = (lane & 1) * 8;
    auto values = [&](const uint8_t *vals, int d, int j) {
        const uint8_t *at = vals + (16 * j + vrow) * ROW + ((4 * d + vch) ^ vx) * 16 + voff;
        const pg_s4 u = pg_read_columns(at), v = pg_read_columns(at + 8 * ROW);
        return __builtin_bit_cast(Frag, pg_s8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
    };

    const uint32_t t_first = t;
    int st = 0;
    if constexpr (BLOCKS) {
        if (t < t_end) store(0, base + t * 64, here != kNoPage);
    }
    for (; t < t_end; t++, st ^= 1) {
        if constexpr (BLOCKS) {
            lds_barrier();      // behind it a stage is whole, and the other one, which was read before it, free
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        auto next = [&]() {
            if (t + 1 >= t_end) return;
            const uint32_t in = (base + (t + 1) * 64 + wave * 16) & (psize - 1);
            here = mine;
            if constexpr (BLOCKS) fetch(here, in);
            else issue(st ^ 1, here, in);
            if (t + 2 < t_end) mine = page_of(base + (t + 2) * 64 + wave * 16);
        };
        auto finish = [&]() {
            if constexpr (BLOCKS) {
                if (t + 1 < t_end) store(st ^ 1, base + (t + 1) * 64, here != kNoPage);
            }
        };
        const uint32_t kb = base + t * 64, ok = pages_of(kb);
        uint8_t *kt_lds = lds + st * STAGE, *vt_lds = kt_lds + 64 * ROW;
        if constexpr (!BLOCKS) {
            if (partly(kb, ok)) clean(vt_lds, kb, ok);
        }
        if (idle || kb >= own.hi || kb + 64 <= own.lo) {
            next();
            finish();
            continue;
        }
        if constexpr (BLOCKS) next();
        const bool edge = kb < own.all_lo || kb + 64 > own.all_hi || ok != 15;

        pg_f16v sc[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[kt][i] = 0.f;
        auto key = [&](int kt, int k) {
            const int row = kt * 32 + l32;
            return *reinterpret_cast<const Frag *>(kt_lds + row * ROW + ((2 * k + hh) ^ (row % (CH < 16 ? CH : 16))) * 16);
        };
        if constexpr (BLOCKS) {
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    pg_f16v acc;
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[i] = 0.f;
                    acc = pg_mfma32<BF>(key(kt, 2 * b), q[2 * b], acc);
                    acc = pg_mfma32<BF>(key(kt, 2 * b + 1), q[2 * b + 1], acc);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const pg_h4 d = *reinterpret_cast<const pg_h4 *>(key_scales + (st * KB + b) * 64 + 32 * kt + 2 * i + 4 * hh);
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[kt][i + e] = fmaf((float)d[e], acc[i + e], sc[kt][i + e]);
                    }
                }
        } else {
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++) sc[kt] = pg_mfma32<BF>(key(kt, k), q[k], sc[kt]);
            // reads four products ahead: left alone the compiler reads a pair, waits and multiplies
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int k = 0; k < 2 * KS - 4; k++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
            next();      // its scalar work while the products run
        }
        // score i of kt is key 32 kt + 8 (i / 4) + 4 hh + i % 4
        if (edge) {
            const uint32_t first = kb + 4 * hh - lo;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const uint32_t sees = (ok >> (2 * kt + i / 8)) & 1 ? span : 0u;
                    sc[kt][i] = first + (32 * kt + 8 * (i / 4) + i % 4) < sees ? sc[kt][i] : -INFINITY;
                }
        }
        Frag p[4], rest[FINE ? 4 : 1];      // 16 keys each
        float sum;
        auto weigh = [&](auto exponent) {
            sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float w = pg_exp2(exponent(sc[j / 2][j % 2 * 8 + e]));
                    sum += w;
                    if constexpr (BF) {
                        p[j][e] = (__bf16)w;
                    } else {
                        const _Float16 h = (_Float16)w;
                        p[j][e] = h;
                        if constexpr (FINE) rest[j][e] = (_Float16)(w - (float)h);
                    }
                }
        };
        const auto near = [&](float s) { return fmaf(s, factor, less); };
        weigh(near);
        if (__any(!(sum <= MOST))) {      // the reference is too small, as at first; or a score is no number
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(sc[kt][i], sc[kt][i + 1]), top);
            const float to = fmaxf(fmaxf(top, __shfl_xor(top, 32, 64)) * factor, m), f = pg_exp2(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= f;
            // A product and its rounding, the reference, are far apart where they are large: the weights are then those of rounded products, and the row comes here in every tile
            const bool far = fabsf(m) > kFar;
            less = far ? -kNothing : kLift - m;
            if (__any(far)) weigh([&](float s) { return far ? pg_apart(s, factor, m) + kLift : near(s); });
            else weigh(near);
        }
        l += sum;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const Frag v = values(vt_lds, d, j);
                if constexpr (FINE) o[d] = pg_mfma32<BF>(v, rest[j], o[d]);
                o[d] = pg_mfma32<BF>(v, p[j], o[d]);
            }
        finish();
    }
    if constexpr (!BLOCKS) {
        float odd = 0.f;      // NaN where one of the results is not finite
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) odd = fmaf(o[d][i], 0.f, odd);
        if (odd != odd) special = 1;
    }
    __syncthreads();
    const bool odd = !BLOCKS && special;
    if (odd) {
        // A row that sees numbers that are not finite has their sum, whatever they weigh (a weight of 0 would have made NaN of an infinity).  Kinds 1 to 3, NaN, inf and -inf: their
        // counts among the keys that a row sees, as a product of ones.
        pg_f16v sums[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) sums[d][i] = 0.f;
        for (t = t_first; t < t_end; t++) {
            const uint32_t kb = base + t * 64, ok = pages_of(kb);
            issue(0, page_of(kb + wave * 16), (kb + wave * 16) & (psize - 1));
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll 1
            for (int kind = 1; kind <= 3; kind++) {
                const float add = kind == 1 ? __builtin_nanf("") : kind == 2 ? INFINITY : -INFINITY;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    pg_f16v n;
#pragma unroll
                    for (int i = 0; i < 16; i++) n[i] = 0.f;
                    for (int j = 0; j < 4; j++) {
                        Frag one;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float w = kb + 4 * hh - lo + (16 * j + 8 * (e / 4) + e % 4) < ((ok >> j) & 1 ? span : 0u) ? 1.f : 0.f;
                            if constexpr (BF) one[e] = (__bf16)w;
                            else one[e] = (_Float16)w;
                        }
                        n = pg_mfma32<BF>(pg_only<BF>(values(lds + 64 * ROW, d, j), kind), one, n);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) sums[d][i] += n[i] > 0.f ? add : 0.f;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = sums[d][i] == 0.f ? o[d][i] : sums[d][i];
    }

    l += __shfl_xor(l, 32, 64);
    const uint32_t r = w0 + l32;
    if (r >= rows) return;
    // register i of d is dimension 32 d + 8 (i / 4) + 4 hh + i % 4
    if (it.parts > 1) {
        const uint64_t at = ((uint64_t)item * a.c.kv_heads + head) * kPagedTileRows + wave * 32 + l32;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4 *>(a.part + at * D + 32 * d + 2 * i + 4 * hh) = make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
        if (hh == 0) {
            a.part_ml[2 * at] = m;
            a.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const uint32_t tk = r / group, h = head * group + (r - tk * group);
    float f = 1.f;
    if (a.sinks) {
        const float sink = a.sinks[h] * 1.44269504088896341f, over = fmaxf(m, sink);
        f = pg_exp2(m - over);
        l = fmaf(l, f, pg_exp2(sink - over + kLift));
    }
    f = l == 0.f ? 0.f : f / l;
    uint16_t *out = static_cast<uint16_t *>(a.out) + (uint64_t)(it.s.row0 + tk) * a.ldo + (uint64_t)h * D;
    const bool half = a.type == LV_F16;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = l == 0.f ? 0.f : o[d][i + e] * (odd ? pg_weight(o[d][i + e], f) : f);
            uint32_t lo2, hi2;
            if (half) {
                lo2 = pg_bits(y[0], true) | (pg_bits(y[1], true) << 16);
                hi2 = pg_bits(y[2], true) | (pg_bits(y[3], true) << 16);
            } else {
                lo2 = pg_bits(y[0], false) | (pg_bits(y[1], false) << 16);
                hi2 = pg_bits(y[2], false) | (pg_bits(y[3], false) << 16);
            }
            *reinterpret_cast<uint2 *>(out + 32 * d + 2 * i + 4 * hh) = make_uint2(lo2, hi2);
        }
}

// ---- the parts of cut items put together -------------------------------------------------------------------------------------------
// Bound by its launch and a chain of loads: lengths, then a row's maxima and results (2.8 us for 32 rows of 4 parts, 4.8 for 2048 of two).
// WAVES waves a row, 4 / WAVES rows a workgroup: four for few rows, which may have many parts; one where there are many rows and most workgroups find nothing to do.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, float lift)
{
    __shared__ float sums[4][D], tops[4][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = wave / WAVES * WAVES;
    const uint32_t heads = a.c.kv_heads * a.deal.group, n = blockIdx.x * (4 / WAVES) + wave / WAVES, row = n / heads, h = n - row * heads;
    PagedItem it{};
    if (row < a.deal.tokens) it = paged_locate<true>(a, row, lane, h % a.deal.group);
    const bool cut = it.any && it.parts > 1;
    if constexpr (WAVES == 4) {
        if (!cut) return;
    }
    const uint32_t group = a.deal.group, kvh = h / group, r = (row - it.s.row0) * group + h % group, in = r - it.tile * a.deal.tile;
    // of a row's parts a wave takes every WAVES-th
    constexpr int V = D >= 64 ? D / 64 : 1;
    const bool mine = lane * V < D;
    float top = kNothing, all = 0.f, y[V];
#pragma unroll
    for (int e = 0; e < V; e++) y[e] = 0.f;
    for (uint32_t p0 = wave - first; cut && p0 < it.parts; p0 += 4 * WAVES) {
        float ms[4], ls[4], v[4][V];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t p = p0 + WAVES * j;
            const uint64_t at = ((uint64_t)min(it.first + min(p, it.parts - 1), a.items - 1) * a.c.kv_heads + kvh) * a.deal.tile + in;
            ms[j] = a.part_ml[2 * at];
            ls[j] = a.part_ml[2 * at + 1];
            if (p >= it.parts) {
                ms[j] = kNothing;
                ls[j] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < V; e++) v[j][e] = mine && p < it.parts ? a.part[at * D + lane * V + e] : 0.f;
        }
        const float big = fmaxf(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), top), f = pg_exp2(top - big);
        top = big;
        float g[4];
        bool lost = f == 0.f && all != 0.f;      // has the weight of something underflowed?
#pragma unroll
        for (int j = 0; j < 4; j++) {
            g[j] = pg_exp2(ms[j] - big);
            lost |= g[j] == 0.f && ls[j] != 0.f;
        }
        all *= f;
        if (__any(lost)) {      // care for what is not finite
#pragma unroll
            for (int e = 0; e < V; e++) {
                y[e] *= pg_weight(y[e], f);
#pragma unroll
                for (int j = 0; j < 4; j++) y[e] = fmaf(v[j][e], pg_weight(v[j][e], g[j]), y[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) {
                y[e] *= f;
#pragma unroll
                for (int j = 0; j < 4; j++) y[e] = fmaf(v[j][e], g[j], y[e]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) all = fmaf(ls[j], g[j], all);
    }
#pragma unroll
    for (int e = 0; e < V; e++)
        if (mine) sums[wave][lane * V + e] = y[e];
    if (lane == 0) {
        tops[wave][0] = top;
        tops[wave][1] = all;
    }
    __syncthreads();
    if (!cut || wave != first || lane >= D / 8) return;
    float big = tops[first][0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) big = fmaxf(big, tops[first + w][0]);
    const float sink = a.sinks ? a.sinks[h] * 1.44269504088896341f : kNothing;
    big = fmaxf(big, sink);
    float total = a.sinks ? pg_exp2(sink - big + lift) : 0.f, z[8];
    bool lost = false;
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const float g = pg_exp2(tops[first + w][0] - big);
        lost |= g == 0.f && tops[first + w][1] != 0.f;
        total = fmaf(tops[first + w][1], g, total);
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = fmaf(sums[first + w][lane * 8 + e], g, z[e]);
    }
    if (lost) {      // once more, with care for what is not finite
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = 0.f;
#pragma unroll 1
        for (int w = 0; w < WAVES; w++) {
            const float g = pg_exp2(tops[first + w][0] - big);
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = fmaf(sums[first + w][lane * 8 + e], pg_weight(sums[first + w][lane * 8 + e], g), z[e]);
        }
    }
    const float f = 1.f / total;
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = total == 0.f ? 0.f : z[e] * f;
    pg_store8(a.out, a.type, (uint64_t)row * a.ldo + (uint64_t)h * D + lane * 8, z);
}

}  // namespace lv
