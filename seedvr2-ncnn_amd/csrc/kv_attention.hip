// Attention of new rows over a key/value cache in pages (gfx950): a sliding
// window and first tokens that stay visible, pages in bf16 or in four bits.
//
// out = sum_k exp(scale q.k - m) v_k / sum_k exp(scale q.k - m) over the keys
// a row sees, in one pass with the running maximum m. The rows of one sequence
// that share a key/value head (its new tokens times the query heads of a
// group) are packed into row tiles; the key tiles that a row tile sees (those
// of the sinks, then those of the window) are dealt to one or several
// workgroups, whose parts kv_merge_kernel joins.
//
// fp32 rows: queries and probabilities are three bf16 pieces (all 24 bits), so
// that products with the cache's values are exact and sums are fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "awa_device.h"
#include "kv_device.h"
#include "kv_kernels.h"

namespace awa
{
namespace
{

using namespace dev;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr int kRowTile = 16;   // rows of kv_rows_kernel's tile
constexpr int kTileRows = 128; // of kv_tile_kernel's
constexpr int kKeyShift = 5;   // keys of both kernels' key tiles
constexpr int kKeyTile = 1 << kKeyShift;
constexpr int kWaves = 4;     // of kv_rows_kernel's workgroup
constexpr int kWideWaves = 8; // where a CU has but one
constexpr int kLongPart = 256; // key tiles of a part

__device__ __forceinline__ float max_xor16(float x)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float sum_xor16(float x)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// x as PIECES bf16 values whose sum is x rounded to 8 PIECES bits.
template <int PIECES>
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&out)[PIECES])
{
#pragma unroll
    for (int e = 0; e < 8; e++)
    {
        float rest = x[e];
#pragma unroll
        for (int i = 0; i < PIECES; i++)
        {
            const __bf16 b = static_cast<__bf16>(rest);
            out[i][e] = b;
            rest -= static_cast<float>(b);
        }
    }
}

// One row of an output accumulator (O^T, 32 features a block) times `by`.
template <typename T, int N>
__device__ __forceinline__ void store_o(T* dst, const f32x16 (&o)[N], float by, int half)
{
#pragma unroll
    for (int d = 0; d < N; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            store4(dst + 32 * d + 8 * g + 4 * half, o[d][4 * g] * by, o[d][4 * g + 1] * by, o[d][4 * g + 2] * by,
                   o[d][4 * g + 3] * by);
}

typedef __attribute__((address_space(3))) char lds_char;
// (Scalar loads: a vector load of a page would wait for the loads to LDS before
// it.)
typedef const __attribute__((address_space(4))) int constant_int;

// Whether eight bf16 values are finite, and the finite ones of them (else 0).
__device__ __forceinline__ bool finite8(const uint4& v)
{
    const unsigned words[4] = {v.x, v.y, v.z, v.w};
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 4; e++)
        most = max(most, max(words[e] & 0x7fffu, (words[e] >> 16) & 0x7fffu));
    return most < 0x7f80u;
}

__device__ __forceinline__ uint4 only_finite8(const uint4& v)
{
    unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
    {
        words[e] = (words[e] & 0x7f80u) == 0x7f80u ? words[e] & 0xffff0000u : words[e];
        words[e] = (words[e] & 0x7f800000u) == 0x7f800000u ? words[e] & 0xffffu : words[e];
    }
    return make_uint4(words[0], words[1], words[2], words[3]);
}

// A part's row and its (maximum, sum): all rows of part 0, of part 1, ..., then
// the pairs. `row`: of part_index.
__device__ __forceinline__ size_t part_index(const KvParts& k, int seq, const KvSequence& s, int token)
{
    return static_cast<size_t>(k.seq_rows > 0 ? static_cast<long long>(seq) * k.seq_rows : s.first) + token;
}

__device__ __forceinline__ float* part_row(const KvAttentionLaunch& p, const KvParts& k, int dim, int part, size_t row,
                                           int head)
{
    const size_t all = static_cast<size_t>(k.rows) * p.heads.d;
    return k.partial + (part * all + row * p.heads.d + head) * dim;
}

__device__ __forceinline__ float* part_stats(const KvAttentionLaunch& p, const KvParts& k, int dim, int part, size_t row,
                                             int head)
{
    const size_t all = static_cast<size_t>(k.rows) * p.heads.d;
    return k.partial + k.splits * all * dim + (part * all + row * p.heads.d + head) * 2;
}

// Whether some row of those from `first` to `last` (spans) may see some key of the
// 16 from `key` on.
__device__ __forceinline__ bool some_row_sees(int key, const KvSpan& first, const KvSpan& last)
{
    return key < last.end && (key + 16 > first.begin || key < last.sinks);
}

// One row tile of 16 rows, one part of its keys: each of four (eight) waves takes
// every fourth (eighth) key tile (32 keys) by itself, with K from memory straight into the MFMA
// operand registers and V through the wave's own LDS, from which it is read
// transposed; the waves' results are joined at the end. Bound by reading the
// cache: the next tile's rows are asked for as soon as this one's registers are
// free. One row over 131072 keys of 20 heads of 128, bf16: 227 us with the join,
// 5.9 TB/s; 32 rows of up to 16384 keys over four bits 166 us, 5.0 TB/s, where
// unpacking the codes shares the vector units with the softmax. (Eight or sixteen
// waves a workgroup where CUs have several, and registers for three or four
// workgroups of bf16 pages a CU were slower, as were chunks of V in an order that
// frees LDS of bank conflicts: 36.5 us to 35.9 for bf16 rows of 16 sequences of
// 8000 keys, 31.2 to 32.3 for fp32 ones.)
//
// S^T = K Q^T (16x16x32): lane (r = lane % 16, g = lane / 16) holds row r's
// scores of keys 4 g + [0, 4) of each 16. Those of two blocks are, in that
// order, the eight values a lane holds of the PV product's operand P^T; V^T is
// read in the same key order. Which features an MFMA takes of a row does not
// matter as long as both operands agree: of 4-bit rows a lane has a quarter,
// one load and one scale.
template <int D, bool F32, bool FOUR, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void kv_rows_kernel(const KvAttentionLaunch p)
{
    constexpr int kPieces = F32 ? 3 : 1;
    constexpr int kChunks = D / 32;
    constexpr int kBlocks = D / 16;
    constexpr int kPitch = D + 16; // V rows in LDS, elements: eight rows' reads touch all banks
    constexpr int kElem = F32 ? 4 : 2;
    constexpr int kVBytes = kKeyTile * kPitch * 2;
    constexpr int kOBytes = kRowTile * D * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[WAVES][kVBytes > kOBytes ? kVBytes : kOBytes];
    __shared__ float stats[WAVES][kRowTile][2];

    const KvView& c = p.cache;
    const int seq = (blockIdx.y + blockIdx.z) % gridDim.y;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15;
    const int g = lane >> 4;
    // (Parts are in the slowest order, the last ones first, which only long
    // sequences have: workgroups go to the XCDs in turn, and with parts in the
    // fastest order one XCD got the first part of every sequence.)
    const int tile = blockIdx.x / c.heads;
    const int head = blockIdx.x - tile * c.heads;
    const int split = p.one.splits - 1 - blockIdx.z;
    const int part_tiles = p.one.part_tiles;

    const KvSequence s = kv_sequence(c, seq);
    if (s.bad && c.status && threadIdx.x == 0)
        atomicOr(c.status, static_cast<int>(s.bad));
    const int rows = s.rows * p.group.d;
    const int row0 = tile * kRowTile;
    if (row0 >= rows)
        return;
    const int last = min(row0 + kRowTile, rows) - 1;
    const int slot0 = s.length - s.rows;
    const KvSpan span_first = kv_span(p.mask, slot0 + kv_divide(row0, p.group), s.length);
    const KvSpan span_last = kv_span(p.mask, slot0 + kv_divide(last, p.group), s.length);
    const KvTiles tiles = kv_tiles(span_first, span_last, kKeyShift);
    const int count = tiles.sinks + tiles.rest;
    if (split * part_tiles >= count && p.one.splits > 1)
    {
        // No keys: the join leaves this part out.
        const int i = row0 + threadIdx.x;
        if (threadIdx.x < kRowTile && i <= last)
        {
            const int t = kv_divide(i, p.group);
            part_stats(p, p.one, D, split, part_index(p.one, seq, s, t), head * p.group.d + i - t * p.group.d)[0] =
                -INFINITY;
        }
        return;
    }
    // (The last one takes all that is left: lengths may pass their bound.)
    const int part_end = split + 1 == p.one.splits ? count : min(count, (split + 1) * part_tiles);

    // This lane's row (rows past the end repeat the last; they are not stored).
    const int row = min(row0 + r, last);
    const int token = kv_divide(row, p.group);
    const int q_head = head * p.group.d + row - token * p.group.d;
    const KvSpan span = kv_span(p.mask, slot0 + token, s.length);
    bf16x8 q[kChunks][kPieces];
    {
        const unsigned char* src =
            p.q.data + static_cast<long long>(s.first + token) * p.q.stride + static_cast<long long>(q_head) * D * kElem;
#pragma unroll
        for (int i = 0; i < kChunks; i++)
        {
            const int feature = FOUR ? D / 4 * g + 8 * i : 32 * i + 8 * g;
            float v[8];
            uint32_t w[8];
            if (F32)
            {
                load_raw8(reinterpret_cast<const float*>(src) + feature, w);
                raw_to_float8<float>(w, v);
            }
            else
            {
                load_raw8(reinterpret_cast<const uint16_t*>(src) + feature, w);
                raw_to_float8<uint16_t>(w, v);
            }
            split_bf16<kPieces>(v, q[i]);
        }
    }

    constant_int* const table = (constant_int*)(c.table + static_cast<long long>(seq) * c.table_stride);
    const int slot_mask = (1 << c.page_shift) - 1;
    unsigned bad = 0;
    // A key tile: its first key, which of its two 16-key blocks are there, and
    // their pool rows (of which there are less than 2^31). (A block behind the
    // last key has the last key's page; it is masked.)
    struct Tile
    {
        int key0;
        unsigned there;
        size_t base[2];
    };
    auto look_up = [&](int i) {
        Tile t;
        t.key0 = (i < tiles.sinks ? i : tiles.begin + i - tiles.sinks) << kKeyShift;
        t.there = 0;
#pragma unroll
        for (int b = 0; b < 2; b++)
        {
            const int key = t.key0 + 16 * b;
            const int page = table[min(key, span_last.end - 1) >> c.page_shift];
            const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(c.pages);
            if (ok && key < span_last.end)
                t.there |= 1u << b;
            // (A page that the tile has no visible key in is not needed.)
            if (!ok && some_row_sees(key, span_first, span_last))
                bad = AWA_KV_BAD_PAGE;
            t.base[b] = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(
                (((ok ? page : 0) * c.heads + head) << c.page_shift) + (key & slot_mask)));
        }
        return t;
    };

    // K: lane r of block b has key 16 b + r. V: kVLanes lanes a row.
    constexpr int kVLanes = FOUR ? D / 32 : D / 8;
    constexpr int kVRows = 64 / kVLanes;
    constexpr int kVLoads = (kKeyTile + kVRows - 1) / kVRows;
    const int v_row = lane / kVLanes;
    const int v_part = lane % kVLanes;
    uint4 k_raw[2][FOUR ? 1 : kChunks], v_raw[kVLoads];
    unsigned k_byte[2], v_byte[kVLoads];
    auto fetch_k = [&](const Tile& t) {
#pragma unroll
        for (int b = 0; b < 2; b++)
        {
            if (FOUR)
            {
                const unsigned char* const at = c.k + t.base[b] * (D / 2) + r * (D / 2) + g * (D / 8);
                if (D == 128)
                    k_raw[b][0] = *reinterpret_cast<const uint4*>(at);
                else
                {
                    const uint2 w = *reinterpret_cast<const uint2*>(at);
                    k_raw[b][0] = make_uint4(w.x, w.y, 0, 0);
                }
                k_byte[b] = c.k_scale[t.base[b] * (D / kKvGroup) + r * (D / kKvGroup) + g * D / 4 / kKvGroup];
            }
            else
            {
                const unsigned char* const at = c.k + t.base[b] * (D * 2) + r * (D * 2) + g * 16;
#pragma unroll
                for (int j = 0; j < kChunks; j++)
                    k_raw[b][j] = *reinterpret_cast<const uint4*>(at + 64 * j);
            }
        }
    };
    auto fetch_v = [&](const Tile& t) {
#pragma unroll
        for (int j = 0; j < kVLoads; j++)
        {
            const int local = j * kVRows + v_row;
            const size_t base = kVRows > 16 ? (local & 16 ? t.base[1] : t.base[0]) : t.base[j * kVRows / 16];
            if (FOUR)
            {
                const unsigned char* const at = c.v + base * (D / 2) + (local & 15) * (D / 2) + v_part * 16;
                v_raw[j] = *reinterpret_cast<const uint4*>(at);
                v_byte[j] = c.v_scale[base * (D / kKvGroup) + (local & 15) * (D / kKvGroup) + v_part];
            }
            else
                v_raw[j] = *reinterpret_cast<const uint4*>(c.v + base * (D * 2) + (local & 15) * (D * 2) + v_part * 16);
        }
    };

    f32x4 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    float row_max = -INFINITY;
    float row_sum = 0.f;
    unsigned char* const v_lds = lds[wave];

    int i = split * part_tiles + wave;
    Tile now{}, next{};
    if (i < part_end)
    {
        now = look_up(i);
        fetch_k(now);
        fetch_v(now);
        next = look_up(min(i + WAVES, part_end - 1));
    }
#pragma unroll 1
    for (; i < part_end; i += WAVES)
    {
        const int key0 = now.key0;
        // Whether every row of the tile sees all its keys.
        const bool whole = now.there == 3u &&
                           ((key0 >= span_last.begin && key0 + kKeyTile <= span_first.end) ||
                            key0 + kKeyTile <= span_first.sinks);
        f32x4 acc[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
        {
            const float unit = FOUR ? four_unit(k_byte[b]) : 0.f;
            acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < kChunks; j++)
            {
                bf16x8 k;
                if (FOUR)
                {
                    const unsigned words[4] = {k_raw[b][0].x, k_raw[b][0].y, k_raw[b][0].z, k_raw[b][0].w};
                    k = __builtin_bit_cast(bf16x8, four_bf16(words[j], unit));
                }
                else
                    k = __builtin_bit_cast(bf16x8, k_raw[b][j]);
#pragma unroll
                for (int e = kPieces - 1; e >= 0; e--)
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[j][e], acc[b], 0, 0, 0);
            }
        }
        // (Behind the last tile the last is fetched again.)
        fetch_k(next);

        // V into LDS; of tiles that some row sees in part, keys that no row sees
        // as zeros.
        bool finite = true;
#pragma unroll
        for (int j = 0; j < kVLoads; j++)
        {
            const int local = j * kVRows + v_row;
            uint4 w[FOUR ? 4 : 1];
            if (FOUR)
            {
                const float unit = four_unit(v_byte[j]);
                const unsigned words[4] = {v_raw[j].x, v_raw[j].y, v_raw[j].z, v_raw[j].w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[e] = four_bf16(words[e], unit);
            }
            else
                w[0] = v_raw[j];
            if (!whole)
            {
                const int key = key0 + local;
                const bool seen = ((now.there >> (local >> 4)) & 1u) && key < span_last.end &&
                                  (key >= span_first.begin || key < span_last.sinks);
#pragma unroll
                for (int e = 0; e < (FOUR ? 4 : 1); e++)
                {
                    w[e] = seen ? w[e] : make_uint4(0, 0, 0, 0);
                    finite = finite && finite8(w[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < (FOUR ? 4 : 1); e++)
                *reinterpret_cast<uint4*>(v_lds + local * kPitch * 2 + v_part * (FOUR ? 64 : 16) + e * 16) = w[e];
        }
        const unsigned there = now.there;
        now = next;
        fetch_v(now);
        next = look_up(min(i + 2 * WAVES, part_end - 1));

        float x[8];
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = acc[e >> 2][e & 3] * p.scale_log2;
        if (!whole)
        {
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const int key = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
                const bool seen = ((there >> (e >> 2)) & 1u) && key < span.end && (key >= span.begin || key < span.sinks);
                x[e] = seen ? x[e] : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            top = fmaxf(top, x[e]);
        top = max_xor32(max_xor16(top));
        if (__any(top > row_max))
        {
            const float m = fmaxf(row_max, top);
            // (Before the first weight there is nothing but what is not finite.)
            const float alpha = row_max == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(row_max - m);
            row_max = m;
            row_sum *= alpha;
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[b][e] *= alpha;
        }
        const float from = row_max == -INFINITY ? 0.f : row_max;
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = __builtin_amdgcn_exp2f(x[e] - from);
        bf16x8 w[kPieces];
        split_bf16<kPieces>(x, w);
#pragma unroll
        for (int e = 0; e < 8; e++)
            row_sum += F32 ? x[e] : static_cast<float>(w[0][e]);

        // A NaN or an infinity among the values: its product with the zero weight
        // of a row that does not see it would be NaN. Those values are added to
        // the rows that see them (weights are positive), and left out below.
        if (!__all(finite))
        {
#pragma unroll 1
            for (int key = 0; key < kKeyTile; key++)
            {
                const int k = key0 + key;
                const bool sees =
                    ((there >> (key >> 4)) & 1u) && k < span.end && (k >= span.begin || k < span.sinks);
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
                {
                    const uint2 v4 =
                        *reinterpret_cast<const uint2*>(v_lds + key * kPitch * 2 + (16 * b + 4 * g) * 2);
                    const float value[4] = {bf16_lo(v4.x), bf16_hi(v4.x), bf16_lo(v4.y), bf16_hi(v4.y)};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[b][e] += sees && !(fabsf(value[e]) < INFINITY) ? value[e] : 0.f;
                }
            }
            for (int j = lane; j < kKeyTile * (D / 8); j += 64)
            {
                uint4* const at = reinterpret_cast<uint4*>(v_lds + j / (D / 8) * kPitch * 2 + j % (D / 8) * 16);
                *at = only_finite8(*at);
            }
        }
        // (A wave's LDS operations are done in their order.)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
        {
            const unsigned char* const at = v_lds + ((4 * g + (r >> 2)) * kPitch + 16 * b + 4 * (r & 3)) * 2;
            const i16x4 lohi[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at)),
                                   __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 16 * kPitch * 2))};
            const bf16x8 a = __builtin_bit_cast(bf16x8, lohi);
#pragma unroll
            for (int e = kPieces - 1; e >= 0; e--)
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, w[e], o[b], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (bad && c.status && lane == 0)
        atomicOr(c.status, static_cast<int>(bad));

    // Join the waves: each lane group holds a part of its row's sum.
    row_sum = sum_xor32(sum_xor16(row_sum));
    float* const mine = reinterpret_cast<float*>(v_lds);
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        *reinterpret_cast<f32x4*>(mine + r * D + 16 * b + 4 * g) = o[b];
    if (g == 0)
    {
        stats[wave][r][0] = row_max;
        stats[wave][r][1] = row_sum;
    }
    __syncthreads();
    constexpr int kPer = kRowTile * D / (WAVES * 64); // features a thread
    const int out_row = threadIdx.x * kPer / D;
    const int f0 = threadIdx.x * kPer % D;
    if (row0 + out_row > last)
        return;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < WAVES; i++)
        m = fmaxf(m, stats[i][out_row][0]);
    const float from = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    float v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++)
        v[e] = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; i++)
    {
        if (stats[i][out_row][0] == -INFINITY)
            continue;
        const float weight = __builtin_amdgcn_exp2f(stats[i][out_row][0] - from);
        sum += weight * stats[i][out_row][1];
        const float* const part = reinterpret_cast<const float*>(lds[i]) + out_row * D + f0;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            v[e] = fmaf(weight, part[e], v[e]);
    }
    const int out_token = kv_divide(row0 + out_row, p.group);
    const int out_head = head * p.group.d + row0 + out_row - out_token * p.group.d;
    if (p.one.splits > 1)
    {
        const size_t at = part_index(p.one, seq, s, out_token);
        float* const dst = part_row(p, p.one, D, split, at, out_head) + f0;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            dst[e] = v[e];
        if (f0 == 0)
            *reinterpret_cast<float2*>(part_stats(p, p.one, D, split, at, out_head)) = make_float2(m, sum);
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    unsigned char* const dst = const_cast<unsigned char*>(p.out.data) + static_cast<long long>(s.first + out_token) * p.out.stride +
                               (static_cast<long long>(out_head) * D + f0) * kElem;
#pragma unroll
    for (int e = 0; e < kPer; e++)
    {
        if (F32)
            reinterpret_cast<float*>(dst)[e] = v[e] * inv;
        else
            reinterpret_cast<__bf16*>(dst)[e] = static_cast<__bf16>(v[e] * inv);
    }
}

// 16 bytes a lane from base + offset to the 1 KB of LDS at `lds` (lane order);
// the kernel waits for it itself. It has no output register.
__device__ __forceinline__ void load_to_lds(const unsigned char* base, uint32_t offset, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
                 : "memory", "m0");
}

// Workgroups go to the XCDs in turn; each has its own L2. Of every eight units
// (a sequence's key/value head) an XCD takes one, so that the workgroups that
// read the same keys at about the same time share an L2; the rest of the units
// is dealt out part by part. Parts (of a unit's row tiles, those with the most
// keys first) come in their order, for the long ones to start first: a period
// of them holds `each` parts of every unit.
struct TileDeal
{
    int units, parts, each, period, periods; // period: items of an XCD
};

__host__ inline TileDeal tile_deal(int units, int parts)
{
    TileDeal d{units, parts, 1, 0, 0};
    while (units % 8 * d.each % 8)
        d.each *= 2;
    d.period = units * d.each / 8;
    if (units % 8 == 0)
        d.period = units / 8;
    d.periods = (parts + d.each - 1) / d.each;
    return d;
}

struct TileItem
{
    int unit; // < 0: none
    int part;
};

__device__ __forceinline__ TileItem tile_item(const TileDeal& d, int block)
{
    const int xcd = block & 7;
    const int j = block >> 3;
    const int q = j / d.period;
    const int k = j - q * d.period;
    const int whole = d.units >> 3;
    TileItem t;
    if (k < whole * d.each)
    {
        t.part = q * d.each + k / whole;
        // (An XCD's workgroups go to its four shader engines in turn: with a
        // multiple of four units, a long sequence would be on one of them.)
        t.unit = (k + (whole & 3 ? 0 : t.part)) % whole * 8 + xcd;
    }
    else
    {
        const int i = (k - whole * d.each) * 8 + xcd;
        const int left = d.units - whole * 8;
        t.unit = whole * 8 + i % left;
        t.part = q * d.each + i / left;
    }
    return t.part < d.parts ? t : TileItem{-1, 0};
}

// The sequence whose parts item `i` is among, by the whole wave: first[s] <= i <
// first[s + 1].
__device__ __forceinline__ int listed_sequence(const int* first, int sequences, int i)
{
    const int lane = threadIdx.x & 63;
    int step = 1, s = 0;
    while (step * 64 < sequences)
        step *= 64;
    for (;; step /= 64)
    {
        const int at = s + (lane + 1) * step;
        s += __popcll(__ballot(at <= sequences && first[min(at, sequences)] <= i)) * step;
        if (step == 1)
            return __builtin_amdgcn_readfirstlane(s);
    }
}

// Numbers the parts of all sequences (KvAttentionLaunch::list), by one workgroup.
// (Sums stay below 2^30; behind what the grid has, they do not matter.)
constexpr int kListThreads = 1024;
__global__ __launch_bounds__(kListThreads) void kv_list_kernel(const KvAttentionLaunch p)
{
    constexpr long long kMost = 1ll << 30;
    __shared__ long long sums[2][kListThreads / 64];
    const KvView& c = p.cache;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long before[2] = {0, 0};
    unsigned bad = 0;
    for (int base = 0; base < c.sequences; base += kListThreads)
    {
        const int seq = base + threadIdx.x;
        long long n[2] = {0, 0};
        if (seq < c.sequences)
        {
            const KvSequence s = kv_sequence(c, seq);
            const int rows = s.rows * p.group.d;
            bad |= s.bad;
            if (rows > kTileRows)
            {
                const int tiles = (rows + kTileRows - 1) / kTileRows, split = min(tiles, p.more.tiles);
                n[0] = tiles - split + static_cast<long long>(split) * p.more.splits;
            }
            else if (rows > 0)
                n[1] = p.one.splits;
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
        {
            const long long own = n[e];
#pragma unroll
            for (int off = 1; off < 64; off *= 2)
            {
                const long long up = __shfl_up(n[e], off, 64);
                n[e] += lane >= off ? up : 0;
            }
            if (lane == 63)
                sums[e][wave] = n[e];
            n[e] -= own;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; e++)
        {
            long long all = 0;
            for (int w = 0; w < kListThreads / 64; w++)
            {
                n[e] += w < wave ? sums[e][w] : 0;
                all += sums[e][w];
            }
            if (seq < c.sequences)
                p.list[e * (c.sequences + 1) + seq] = static_cast<int>(min(kMost, before[e] + n[e]));
            before[e] = min(kMost, before[e] + all);
        }
        __syncthreads();
    }
    if (threadIdx.x < 2)
        p.list[threadIdx.x * (c.sequences + 1) + c.sequences] = static_cast<int>(before[threadIdx.x]);
    if (bad && c.status)
        atomicOr(c.status, static_cast<int>(bad));
}

// A tile of 128 rows, 32 a wave; key tiles of 32 go through LDS, which all
// waves read. Bound by the matrix cores, next to them by the softmax's vector
// instructions, and by power: the clock falls to about 1.75 GHz. Three workgroups
// share a CU (two of fp32 rows, whose queries take three times the registers), so
// that one's softmax, waits and edges run beside the others' products: nothing
// else of the loop overlaps by itself, and schedules within a wave gained less.
// 16384 rows of 20 heads, 128 features, causal: 1300 us so (1.04 PFLOP/s; a matrix
// product of 8192^3 reaches 1.2), the matrix cores and the vector units busy for
// somewhat more than half of it each, LDS for a third. Two workgroups that
// take the scores of the next block beside a block's softmax: 1440 us; one such
// of eight waves, whose barriers keep them in step: 1557; four waves of 64 rows,
// which read half the operands but leave a matrix core one wave to be fed by:
// 1834. Without its loads of keys and values the loop would take 1183 us, without
// the exponentials 1244, without half of its LDS reads 1270, with bank conflicts
// that double the LDS cycles 1318: no single part bounds it.
//
// S^T = K Q^T (32x32x16): lane (col = lane % 32, half = lane / 32) holds row
// col's scores of keys 8 (i / 4) + 4 half + i % 4, i < 16; eight of them in a row
// are, in that order, what the lane holds of the PV product's operand P^T, and
// V^T is read in the same key order.
template <int D, bool F32, bool FOUR>
__global__ __launch_bounds__(256, F32 ? 2 : 3) void kv_tile_kernel(const KvAttentionLaunch p, const TileDeal deal)
{
    constexpr int kPieces = F32 ? 3 : 1;
    constexpr int kRows = kTileRows;
    constexpr int kThreads = 256;
    constexpr int kKeys = kKeyTile;
    constexpr int kC = D / 16;
    constexpr int kDb = D / 32;
    constexpr int kRowBytes = D * 2;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kRowChunks = kRowBytes / 16;
    constexpr int kElem = F32 ? 4 : 2;
    constexpr float kGrow = 8.f;
    // Keys and values of this tile and the next.
    __shared__ __attribute__((aligned(1024))) unsigned char k_lds[2][kTileBytes];
    __shared__ __attribute__((aligned(1024))) unsigned char v_lds[2][kTileBytes];
    // The last tile with values that are not finite.
    __shared__ int raw_tile;

    const KvView& c = p.cache;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31;
    const int half = lane >> 5;
    TileItem item = tile_item(deal, blockIdx.x);
    if (item.unit < 0)
        return;
    int seq = 0, head = item.unit;
    if (p.listed)
    {
        const int longer = __builtin_amdgcn_readfirstlane(p.list[c.sequences]);
        const int* const first = p.list + (item.part < longer ? 0 : c.sequences + 1);
        item.part -= item.part < longer ? 0 : longer;
        if (item.part >= __builtin_amdgcn_readfirstlane(first[c.sequences]))
            return;
        seq = listed_sequence(first, c.sequences, item.part);
        item.part -= __builtin_amdgcn_readfirstlane(first[seq]);
    }
    else
    {
        seq = item.unit / c.heads;
        head = item.unit - seq * c.heads;
    }

    const KvSequence s = kv_sequence(c, seq);
    if (s.bad && c.status && tid == 0)
        atomicOr(c.status, static_cast<int>(s.bad));
    const int rows = s.rows * p.group.d;
    const bool one = rows <= kRows;
    const int part_tiles = one ? p.one.part_tiles : p.more.part_tiles;
    // Row tiles from the end, which see the most keys; unless listed, those of all
    // sequences in step, so that the longest sequence's come first. The first of
    // a sequence, which come last, may alone be split.
    const int tiles_all = one ? 1 : p.listed ? (rows + kRows - 1) / kRows : p.tiles;
    const int whole = one ? 0 : max(tiles_all - p.more.tiles, 0);
    const int splits = item.part < whole ? 1 : one ? p.one.splits : p.more.splits;
    const int part = item.part < whole ? item.part : item.part - whole;
    const int tile = (item.part < whole ? tiles_all : tiles_all - whole) - 1 - part / splits;
    const int split = part % splits;
    const int row0 = tile * kRows;
    if (tile < 0 || row0 >= rows)
        return;
    const int slot0 = s.length - s.rows;
    auto span_of = [&](int row) { return kv_span(p.mask, slot0 + kv_divide(row, p.group), s.length); };
    const KvSpan first = span_of(row0);
    const KvSpan last = span_of(min(row0 + kRows, rows) - 1);

    // This wave's rows (past the end: the last row again, not stored).
    const int wave_row0 = row0 + wave * 32;
    const bool active = wave_row0 < rows;
    const KvSpan w_first = span_of(min(wave_row0, rows - 1));
    const KvSpan w_last = span_of(min(wave_row0 + 32, rows) - 1);
    // (Worked out again where it is needed: registers are what limits how many
    // workgroups a CU holds. The lane is hidden from the compiler for that.)
    struct Row
    {
        int token, head;
    };
    auto my_row = [&]() {
        int l = lane;
        asm volatile("" : "+v"(l));
        const int r = min(wave_row0 + (l & 31), rows - 1);
        const int token = kv_divide(r, p.group);
        return Row{token, head * p.group.d + r - token * p.group.d};
    };
    bf16x8 q[kC][kPieces];
    // (Not zero, whose product with the -inf of a masked score is NaN.)
    const float scale = fmaxf(fabsf(p.scale_log2), 1e-37f);
    {
        const Row row = my_row();
        const unsigned char* src = p.q.data + static_cast<long long>(s.first + row.token) * p.q.stride +
                                   static_cast<long long>(row.head) * D * kElem;
#pragma unroll
        for (int i = 0; i < kC; i++)
        {
            float v[8];
            uint32_t w[8];
            if (F32)
            {
                load_raw8(reinterpret_cast<const float*>(src) + 16 * i + 8 * half, w);
                raw_to_float8<float>(w, v);
            }
            else
            {
                load_raw8(reinterpret_cast<const uint16_t*>(src) + 16 * i + 8 * half, w);
                raw_to_float8<uint16_t>(w, v);
            }
            if (p.scale_log2 < 0.f)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = -v[e];
            split_bf16<kPieces>(v, q[i]);
        }
    }

    const KvTiles tiles = kv_tiles(first, last, kKeyShift);
    const int t_count = tiles.sinks + tiles.rest;
    if (split * part_tiles >= t_count && splits > 1)
    {
        const Row row = my_row();
        if (half == 0 && wave_row0 + col < rows)
        {
            const KvParts& k = one ? p.one : p.more;
            part_stats(p, k, D, split, part_index(k, seq, s, row.token), row.head)[0] = -INFINITY;
        }
        return;
    }
    const int t_begin = split * part_tiles;
    const int t_end = split + 1 == splits ? t_count : min(t_count, t_begin + part_tiles);

    // Of every tile a wave loads half a 16-key block; of 4-bit pages a block's
    // keys or values.
    constexpr int kLoadRows = FOUR ? 16 : kKeys / 4;
    const int load_block = FOUR ? wave & 1 : wave >> 1;
    const int load_row = FOUR ? 16 * load_block : wave * kLoadRows;
    constant_int* const table = (constant_int*)(c.table + static_cast<long long>(seq) * c.table_stride);
    const int slot_mask = (1 << c.page_shift) - 1;
    auto tile_key = [&](int t) {
        t = min(t, t_end - 1);
        return (t < tiles.sinks ? t : tiles.begin + t - tiles.sinks) << kKeyShift;
    };
    // The pages of a tile's two 16-key blocks, read a tile ahead. (A block behind
    // the last key has the last key's page; it is masked.)
    struct Pages
    {
        int at[2];
    };
    auto pages_of = [&](int key0) {
        return Pages{{table[min(key0, last.end - 1) >> c.page_shift],
                      table[min(key0 + 16, last.end - 1) >> c.page_shift]}};
    };
    // Which blocks have no page of the pool.
    auto missing = [&](const Pages& pages) {
        return static_cast<unsigned>(static_cast<unsigned>(pages.at[0]) >= static_cast<unsigned>(c.pages)) |
               static_cast<unsigned>(static_cast<unsigned>(pages.at[1]) >= static_cast<unsigned>(c.pages)) << 1;
    };
    // The pool row of the wave's first row of the tile (pools have less than 2^31
    // rows).
    auto pool_row_of = [&](int key0, const Pages& pages, unsigned none) {
        const int page = (none >> load_block) & 1u ? 0 : load_block == 0 ? pages.at[0] : pages.at[1];
        return static_cast<size_t>(static_cast<unsigned>(__builtin_amdgcn_readfirstlane(
            ((page * c.heads + head) << c.page_shift) + ((key0 + load_row) & slot_mask))));
    };

    // Where a 16-byte chunk of a row lies in LDS: chunks are permuted so that
    // both operands' reads touch all 64 banks (K: 16 rows, one chunk each; V: four
    // rows, two chunks each).
    auto k_chunk = [](int r, int chunk) { return chunk ^ (D == 128 ? r & 15 : (r >> 1) & 7); };
    auto v_chunk = [](int r, int chunk) { return chunk ^ (D == 128 ? (r & 3) << 2 : (r & 2) << 1); };
    constexpr int kLoads = (kLoadRows * kRowBytes + 1023) / 1024; // loads of 1 KB
    const uint32_t lds_k = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char*)k_lds));
    const uint32_t lds_v = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char*)v_lds));
    const int l_row = lane / kRowChunks; // of the first KB; of KB j: + j * (64 / kRowChunks)
    auto load = [&](size_t pool_row, int slot) {
        const unsigned char* const k = c.k + pool_row * kRowBytes;
        const unsigned char* const v = c.v + pool_row * kRowBytes;
#pragma unroll
        for (int j = 0; j < kLoads; j++)
        {
            const int r = j * (64 / kRowChunks) + l_row;
            const uint32_t at = slot * kTileBytes + load_row * kRowBytes + j * 1024;
            load_to_lds(k + j * 1024, l_row * kRowBytes + k_chunk(load_row + r, lane % kRowChunks) * 16, lds_k + at);
            load_to_lds(v + j * 1024, l_row * kRowBytes + v_chunk(load_row + r, lane % kRowChunks) * 16, lds_v + at);
        }
    };
    // 4-bit pages: two waves load a 16-key block of keys each, two of values, a
    // lane 32 features of a row, in registers until they go to LDS as bf16. (Of
    // 64 features half the lanes suffice. Lanes are dealt out so that eight in a
    // row write to all banks.)
    constexpr int kGroups = D / 32;
    const bool f_value = wave >= 2;
    const int f_row = D == 128 ? ((lane >> 1) & 3) + (lane >> 4) * 4
                               : ((lane >> 1) & 3) * 2 + ((lane >> 3) & 1) + ((lane >> 4) & 1) * 8;
    const int f_group = D == 128 ? (lane & 1) + ((lane >> 3) & 1) * 2 : lane & 1;
    const uint32_t f_from = f_row * kGroups + f_group;
    // Where a lane's four chunks go: chunk j at f_at ^ 16 j.
    uint32_t f_at;
    {
        const int r = load_row + f_row;
        const int low = D == 128 ? r & 3 : (r >> 1) & 3;
        f_at = r * kRowBytes + ((f_value ? v_chunk(r, 4 * f_group) : k_chunk(r, 4 * f_group)) & ~3) * 16 + low * 16;
    }
    uint4 codes;
    unsigned byte;
    auto load_four = [&](size_t pool_row) {
        codes = *reinterpret_cast<const uint4*>((f_value ? c.v : c.k) + pool_row * (D / 2) + f_from * 16);
        byte = ((f_value ? c.v_scale : c.k_scale) + pool_row * kGroups)[f_from];
    };
    auto store_four = [&](int slot) {
        if (lane >= 16 * kGroups)
            return;
        const float unit = four_unit(byte);
        unsigned words[4] = {codes.x, codes.y, codes.z, codes.w};
        if (f_value)
        {
            // (The swizzle of V leaves the low bits of a chunk; written in order,
            // four rows' chunks would share their banks.)
#pragma unroll
            for (int b = 1; b <= 2; b++)
            {
                const bool swap = f_at & (16 * b);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (!(j & b))
                    {
                        const unsigned x = words[j], y = words[j + b];
                        words[j] = swap ? y : x;
                        words[j + b] = swap ? x : y;
                    }
            }
        }
        unsigned char* const dst = f_value ? v_lds[slot] : k_lds[slot];
#pragma unroll
        for (int j = 0; j < 4; j++)
            *reinterpret_cast<uint4*>(dst + (f_at ^ (16 * j))) = four_bf16(words[j], unit);
    };

    f32x16 o[kDb];
#pragma unroll
    for (int d = 0; d < kDb; d++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            o[d][i] = 0.f;
    // (Finite, so that no difference is NaN; nothing that is weighed is below.)
    constexpr float kNoMax = -1.5e38f;
    float row_max = kNoMax, row_sum = 0.f;
    bf16x8 w[2][kPieces]; // a block's weights

    bf16x8 ka[kC], va[2][kDb];
    auto read_k = [&](const unsigned char* k) {
#pragma unroll
        for (int i = 0; i < kC; i++)
            ka[i] = *reinterpret_cast<const bf16x8*>(k + col * kRowBytes + k_chunk(col, 2 * i + half) * 16);
    };
    auto read_v = [&](const unsigned char* v) {
        const int g = (lane >> 4) & 1;
        const int r = lane & 15;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int d = 0; d < kDb; d++)
            {
                const unsigned char* const at = v + (16 * j + 4 * half + (r >> 2)) * kRowBytes +
                                                v_chunk(r >> 2, 4 * d + 2 * g + ((r & 3) >> 1)) * 16 + (r & 1) * 8;
                const i16x4 lohi[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at)),
                                       __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 8 * kRowBytes))};
                va[j][d] = __builtin_bit_cast(bf16x8, lohi);
            }
    };
    auto qk = [&](f32x16& x) {
#pragma unroll
        for (int i = 0; i < 16; i++)
            x[i] = 0.f;
#pragma unroll
        for (int i = 0; i < kC; i++)
#pragma unroll
            for (int e = kPieces - 1; e >= 0; e--)
                x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[i], q[i][e], x, 0, 0, 0);
    };
    auto pv = [&]() {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = kPieces - 1; e >= 0; e--)
#pragma unroll
                for (int d = 0; d < kDb; d++)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[j][d], w[j][e], o[d], 0, 0, 0);
    };
    auto top_of = [&](const f32x16& x) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; i++)
            top = fmaxf(top, x[i]);
        return max_xor32(top);
    };
    // Weights from scores.
    auto weigh = [&](const f32x16& x) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; i++)
            y[i] = __builtin_amdgcn_exp2f(fmaf(x[i], scale, -row_max));
#pragma unroll
        for (int j = 0; j < 2; j++)
        {
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                z[e] = y[8 * j + e];
            split_bf16<kPieces>(z, w[j]);
            if (F32)
            {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    row_sum += z[e];
            }
            else
            {
                const bf16x2 ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
                for (int e = 0; e < 4; e++)
                {
                    const bf16x2 pair = {w[j][0][2 * e], w[j][0][2 * e + 1]};
                    row_sum = __builtin_amdgcn_fdot2_f32_bf16(pair, ones, row_sum, false);
                }
            }
        }
    };
    // A tile's values that are not finite, to the rows that see them; the tile
    // then holds zeros for them (a product with the zero weight of a row that
    // does not see them would be NaN). Weights are positive, so what they weigh
    // does not matter.
    auto add_raw = [&](const unsigned char* v, int key0, unsigned none) {
        const KvSpan span = kv_span(p.mask, slot0 + my_row().token, s.length);
#pragma unroll 1
        for (int key = 0; key < kKeys; key++)
        {
            const int k = key0 + key;
            const bool sees = !((none >> (key >> 4)) & 1u) && k < span.end && (k >= span.begin || k < span.sinks);
#pragma unroll
            for (int d = 0; d < kDb; d++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                {
                    const uint2 v4 =
                        *reinterpret_cast<const uint2*>(v + key * kRowBytes + v_chunk(key, 4 * d + g) * 16 + half * 8);
                    const float value[4] = {bf16_lo(v4.x), bf16_hi(v4.x), bf16_lo(v4.y), bf16_hi(v4.y)};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[d][4 * g + e] += sees && !(fabsf(value[e]) < INFINITY) ? value[e] : 0.f;
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };

    auto wait = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // (LDS alone: the loads of the next tile go on.)
    auto wait_lds = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // The first keys of this tile and the next, the next one's pages, and which
    // blocks of this tile have none.
    int key_now = 0, key_next = 0;
    Pages pages_next{};
    unsigned none = 0;
    if (t_begin < t_end)
    {
        if (tid == 0)
            raw_tile = -1;
        key_now = tile_key(t_begin);
        key_next = tile_key(t_begin + 1);
        const Pages pages = pages_of(key_now);
        pages_next = pages_of(key_next);
        none = missing(pages);
        const size_t row_now = pool_row_of(key_now, pages, none);
        if (FOUR)
            load_four(row_now);
        else
            load(row_now, 0);
    }
#pragma unroll 1
    for (int t = t_begin; t < t_end; t++)
    {
        const int slot = (t - t_begin) & 1;
        unsigned char* const k_tile = k_lds[slot];
        unsigned char* const v_tile = v_lds[slot];
        if (FOUR)
            store_four(slot);
        // This tile is there, and all waves are done with the one before.
        // (Behind the last tile the last is loaded again.)
        wait();
        const unsigned none_next = missing(pages_next);
        const size_t row_next = pool_row_of(key_next, pages_next, none_next);
        if (FOUR)
            load_four(row_next);
        else
            load(row_next, 1 - slot);
        const int key_third = tile_key(t + 2);
        pages_next = pages_of(key_third);
        bool edge = false;
        // Tiles that some row sees in part. What no row of the workgroup sees
        // becomes zeros, and so do values that are not finite.
        if (none != 0u ||
            !((key_now >= last.begin && key_now + kKeys <= first.end) || key_now + kKeys <= first.sinks))
        {
            edge = none != 0u || !((key_now >= w_last.begin && key_now + kKeys <= w_first.end) ||
                                   key_now + kKeys <= w_first.sinks);
            // (A page that the tile has no visible key in is not needed.)
            if (((none & 1u) && some_row_sees(key_now, first, last)) ||
                ((none & 2u) && some_row_sees(key_now + 16, first, last)))
                if (c.status && tid == 0)
                    atomicOr(c.status, AWA_KV_BAD_PAGE);
            uint4* const v = reinterpret_cast<uint4*>(v_tile);
            constexpr int kMine = kKeys * kRowChunks / kThreads;
            bool fine = true;
#pragma unroll
            for (int j = 0; j < kMine; j++)
            {
                const int i = tid + j * kThreads;
                const int k = key_now + i / kRowChunks;
                if (!((none >> (i / kRowChunks >> 4)) & 1u) && k < last.end && (k >= first.begin || k < last.sinks))
                    fine = fine && finite8(v[i]);
                else
                    v[i] = make_uint4(0, 0, 0, 0);
            }
            if (!fine)
                raw_tile = t;
            wait_lds();
            if (raw_tile == t)
            {
                if (active)
                    add_raw(v_tile, key_now, none);
                wait_lds();
#pragma unroll
                for (int j = 0; j < kMine; j++)
                    v[tid + j * kThreads] = only_finite8(v[tid + j * kThreads]);
                wait_lds();
            }
        }
        if (active)
        {
            read_k(k_tile);
            f32x16 x;
            qk(x);
            float top = top_of(x) * scale;
            if (edge)
            {
                const KvSpan span = kv_span(p.mask, slot0 + my_row().token, s.length);
                const int key0 = key_now + 4 * half;
                const int end = span.end - key0, begin = span.begin - key0, sinks = span.sinks - key0;
#pragma unroll
                for (int i = 0; i < 16; i++)
                {
                    const int key = 8 * (i >> 2) + (i & 3);
                    const bool page = !((none >> (i >> 3)) & 1u);
                    x[i] = page & (key < end) & ((key >= begin) | (key < sinks)) ? x[i] : -INFINITY;
                }
                top = top_of(x) * scale;
            }
            if (__any(top > row_max + kGrow))
            {
                const float m = fmaxf(row_max, top);
                // (Before the first weight there is nothing but what is not finite.)
                const float alpha = row_max == kNoMax ? 1.f : __builtin_amdgcn_exp2f(row_max - m);
                row_max = m;
                row_sum *= alpha;
#pragma unroll
                for (int d = 0; d < kDb; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[d][i] *= alpha;
            }
            read_v(v_tile);
            weigh(x);
            pv();
        }
        key_now = key_next;
        key_next = key_third;
        none = none_next;
    }
    // No load of this wave may be on its way into LDS when it ends.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const float sum = sum_xor32(row_sum);
    if (wave_row0 + col >= rows)
        return;
    const Row row = my_row();
    if (splits > 1)
    {
        const KvParts& k = one ? p.one : p.more;
        const size_t at = part_index(k, seq, s, row.token);
        store_o(part_row(p, k, D, split, at, row.head), o, 1.f, half);
        if (half == 0)
            *reinterpret_cast<float2*>(part_stats(p, k, D, split, at, row.head)) =
                make_float2(sum == 0.f ? -INFINITY : row_max, sum);
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    unsigned char* const dst = const_cast<unsigned char*>(p.out.data) +
                               static_cast<long long>(s.first + row.token) * p.out.stride +
                               static_cast<long long>(row.head) * D * kElem;
    if (F32)
        store_o(reinterpret_cast<float*>(dst), o, inv, half);
    else
        store_o(reinterpret_cast<uint16_t*>(dst), o, inv, half);
}

// Joins the parts of a row: M = max m_i, out = sum 2^(m_i - M) o_i / sum
// 2^(m_i - M) l_i, in an order that the number of parts gives; parts without a
// key are left out. 16 lanes hold a row: with GROUPS 1 a wave takes four rows of
// at most 16 parts, with 4 it takes the parts of one, at most 64, in four. All
// parts' maxima and sums come with one load, their rows with independent ones,
// eight at a time.
// Bound by latency where rows are few: 20 rows of 6 parts 4.4 us, of 64 parts 6.2
// (a wave a row, eight parts at a time: 4.2 and 8.8); by memory where they are
// many: 28160 rows of three parts 13.1 us, 4.5 TB/s (a wave a row 18.8).
template <int D, bool F32, int GROUPS>
__global__ __launch_bounds__(256) void kv_merge_kernel(const KvAttentionLaunch p)
{
    constexpr int kPer = D / 16;      // features a lane
    constexpr int kRows = 4 / GROUPS; // rows of a wave
    constexpr int kBatch = 8;
    const KvSequence s = kv_sequence(p.cache, blockIdx.y);
    const bool more = !p.few && s.rows * p.group.d > kTileRows;
    const KvParts k = more ? p.more : p.one;
    if (k.splits == 1)
        return;
    const int lane = threadIdx.x & 15;
    const int group = (threadIdx.x >> 4) & 3;
    const int first_part = GROUPS == 1 ? 0 : group;
    // (Rows of tiles that are not split are there already.)
    const int split_rows = more ? p.more.tiles * kTileRows : kTileRows;
    const int rows = min(s.rows, kv_divide(split_rows - 1, p.group) + 1) * p.heads.d;
    for (int i0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows; i0 < rows; i0 += gridDim.x * 4 * kRows)
    {
        // (Past the last row: that one again, not stored.)
        const int i = min(i0 + (GROUPS == 1 ? group : 0), rows - 1);
        const int token = kv_divide(i, p.heads);
        const int head = i - token * p.heads.d;
        if (token * p.group.d + head - kv_divide(head, p.group) * p.group.d >= split_rows)
            continue;
        const size_t row = part_index(k, blockIdx.y, s, token);
        const int mine_part = lane * GROUPS + first_part;
        const float2 mine = mine_part < k.splits
                                ? *reinterpret_cast<const float2*>(part_stats(p, k, D, mine_part, row, head))
                                : make_float2(-INFINITY, 0.f);
        float m = mine.x;
#pragma unroll
        for (int off = 1; off < 16 * GROUPS; off *= 2)
            m = fmaxf(m, __shfl_xor(m, off, 64));
        const bool has_keys = mine.x != -INFINITY;
        // (< 0: no keys.)
        const float weight = has_keys ? __builtin_amdgcn_exp2f(mine.x - m) : -1.f;
        float sum = has_keys ? weight * mine.y : 0.f;
#pragma unroll
        for (int off = 1; off < 16 * GROUPS; off *= 2)
            sum += __shfl_xor(sum, off, 64);
        float v[kPer];
#pragma unroll
        for (int e = 0; e < kPer; e++)
            v[e] = 0.f;
#pragma unroll 1
        for (int t = 0; t < 16 && t * GROUPS < k.splits; t += kBatch)
        {
            float4 part[kBatch][kPer / 4];
            float by[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; b++)
            {
                by[b] = __shfl(weight, t + b, 16);
                const bool there = !(by[b] < 0.f);
                const float4* const src = reinterpret_cast<const float4*>(
                    part_row(p, k, D, (t + b) * GROUPS + first_part, row, head) + lane * kPer);
#pragma unroll
                for (int e = 0; e < kPer / 4; e++)
                    part[b][e] = there ? src[e] : make_float4(0.f, 0.f, 0.f, 0.f);
                by[b] = there ? by[b] : 0.f;
            }
#pragma unroll
            for (int b = 0; b < kBatch; b++)
#pragma unroll
                for (int e = 0; e < kPer / 4; e++)
                {
                    v[4 * e] = fmaf(by[b], part[b][e].x, v[4 * e]);
                    v[4 * e + 1] = fmaf(by[b], part[b][e].y, v[4 * e + 1]);
                    v[4 * e + 2] = fmaf(by[b], part[b][e].z, v[4 * e + 2]);
                    v[4 * e + 3] = fmaf(by[b], part[b][e].w, v[4 * e + 3]);
                }
        }
        if (GROUPS > 1)
#pragma unroll
            for (int e = 0; e < kPer; e++)
            {
                v[e] += __shfl_xor(v[e], 16, 64);
                v[e] += __shfl_xor(v[e], 32, 64);
            }
        if (GROUPS > 1 ? group != 0 : i0 + group >= rows)
            continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        unsigned char* const dst = const_cast<unsigned char*>(p.out.data) +
                                   static_cast<long long>(s.first + token) * p.out.stride +
                                   (static_cast<long long>(head) * D + lane * kPer) * (F32 ? 4 : 2);
#pragma unroll
        for (int e = 0; e < kPer; e += 4)
        {
            if (F32)
                store4(reinterpret_cast<float*>(dst) + e, v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv);
            else
                store4(reinterpret_cast<uint16_t*>(dst) + e, v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv);
        }
    }
}

} // namespace

namespace
{

// What workgroups of kv_tile_kernel take, measured, in us.
struct TileTimes
{
    double alone; // a key tile, of one that has a CU to itself
    double full;  // of a CU's full set of them side by side
    int set;      // in a full set
    double join;  // writing and reading a part again

    TileTimes(const KvAttentionLaunch& p, long long block_rows)
    {
        const bool half = p.head_dim == 64;
        alone = (p.f32 ? 1.35 : p.four ? 1.0 : 0.75) * (half ? 0.85 : 1.0);
        full = (p.f32 ? 1.8 : p.four ? 1.7 : 1.55) * (half ? 0.9 : 1.0);
        set = p.f32 ? (half && !p.four ? 3 : 2) : half ? 4 : 3;
        join = 0.045 * std::min(block_rows, static_cast<long long>(kTileRows)) / kTileRows * p.head_dim / 128;
    }
};

struct Split
{
    long long n;
    double time;
};

// Parts of a row tile of 128 rows with the least time for `blocks` of them, which
// see `count` key tiles on the average: a CU takes one full set of workgroups
// after the other, and of the last one it has a part. 8 heads of 128 over 8000
// keys (us): 8 workgroups 198, split 28; 64 (1024 rows) 191, split 58. 20 heads:
// 220 (1408 rows over 31408 keys) 728, in three parts 504; 320 (2048 over 8048)
// 218, in two 204; 460 265, in two 322; 100 (640 over 640) 26, in two 31.
Split tile_splits(const TileTimes& c, long long blocks, double count)
{
    const auto time = [&](long long n) {
        const double each = blocks * n / 256.0; // of a CU
        const double sets = std::floor(each / c.set), left = each - sets * c.set;
        double t = sets * c.full;
        if (left > 0)
            t += sets > 0 ? 0.65 * c.alone + left * (c.full - 0.65 * c.alone) / c.set
                          : c.alone + std::max(0.0, left - 1) * (c.full - c.alone) / (c.set - 1);
        return t * count / n + (n > 1 ? 3 + c.join * blocks * n : 0);
    };
    Split s{1, time(1)};
    double best = 0.95 * s.time;
    for (long long n = 2; n <= 64 && n * 4 <= count; n++)
        if (time(n) < best)
        {
            best = time(n);
            s = {n, best};
        }
    return s;
}

// The same where only the first `tiles` row tiles of each of `units` are split,
// which start last: the others fill whole sets, and the parts of these what is
// left. n 1: none takes less time than `best`. 20 heads of 128 (us, without and
// with): 5000 rows over 11000 keys 516, 433; 5760 over 11760 keys of four bits 721,
// 547; 32/8 heads, 3500 over 15500: 869, 751.
struct FirstSplit
{
    long long n;
    int tiles;
};

FirstSplit first_splits(const TileTimes& c, long long blocks, long long units, int tiles, double count, double best)
{
    FirstSplit s{1, 0};
    best *= 0.95;
    const long long places = 256ll * c.set;
    for (long long sets = std::max(1ll, blocks / places - 1); sets * places < blocks && sets <= blocks / places; sets++)
    {
        const long long first = (blocks - sets * places + units - 1) / units;
        if (first >= tiles)
            continue;
        const double left = static_cast<double>(blocks - sets * places) / places;
        for (long long n = 2; n <= 12 && n * 4 <= count; n++)
        {
            const double time =
                ((sets + left) * c.full + 0.5 * c.alone / n) * count + 3 + c.join * units * first * n;
            if (time < best)
            {
                best = time;
                s = {n, static_cast<int>(first)};
            }
        }
    }
    return s;
}

} // namespace

void kv_attention_deal(KvAttentionLaunch& p, int max_length)
{
    const KvView& c = p.cache;
    const int group = p.group.d;
    const long long rows = static_cast<long long>(c.max_rows) * group;
    // Each tile of 16 rows reads the keys for itself. 16 sequences of 8000 keys,
    // 8 heads of 128 and as many rows (us), tiles of 16 and of 128:
    //   bf16: 16 rows 99, 99; 32 rows 155, 100. One of 4000: 16 rows 15, 17.
    //   four bits, which a tile of 128 unpacks into LDS: 16 rows 38, 90; 32 rows
    //   60, 92; 48 rows 82, 96; 64 rows 108, 97.
    p.few = rows <= (p.four ? 3 : 1) * kRowTile;
    const int tile_rows = p.few ? kRowTile : kTileRows;
    p.tiles = static_cast<int>((rows + tile_rows - 1) / tile_rows);
    // Key tiles that a row tile may see.
    long long keys = max_length;
    if (p.mask.window > 0)
        keys = std::min(keys, static_cast<long long>(p.mask.window) + p.mask.sinks + p.mask.block +
                                  std::min(c.max_rows, tile_rows / group + 1));
    const long long count = (keys >> kKeyShift) + 2;
    const auto parts = [&](long long splits) {
        KvParts k{};
        k.splits = static_cast<int>(std::max(1ll, std::min({splits, count, 64ll})));
        k.part_tiles = static_cast<int>((count + k.splits - 1) / k.splits);
        k.tiles = p.tiles;
        k.rows = c.total_rows;
        return k;
    };
    // Few workgroups at the end would have the card to themselves: lengths may
    // differ, so parts are not longer than this. One row each over 99 sequences of
    // 2000 keys and one of 131072, 8 heads (us), parts of 16384, 8192 and 4096
    // keys at most: 317, 305, 282 (450 unsplit); over 127 of 4096 beside a chunk of
    // 1024 rows: 439, 441, 488; over 64 of 16384: 722, 719, 719.
    const long long least = (count + kLongPart - 1) / kLongPart;
    if (p.few)
    {
        // The split with the least time, in key tiles of a workgroup: rounds of
        // workgroups (two to four a CU, by their registers), each with its start
        // and its part, and the join. (A join that counts half, twice or four times
        // as much changes calls of 700 to 6000 keys by -1 to 7 us.)
        const long long blocks = static_cast<long long>(p.tiles) * c.heads * c.sequences;
        const long long slots = 256 * (p.head_dim == 64 ? 4 : p.four ? 3 : 2);
        long long best = -1, splits = 1;
        for (long long n = std::min(least, 64ll); n <= 64 && n <= count; n++)
        {
            const long long part = (count + n - 1) / n;
            if (n > 1 && part < kWaves)
                break;
            const long long time = (blocks * n + slots - 1) / slots * (part + 8) + (n > 1 ? 16 + n / 4 : 0);
            if (best < 0 || time < best)
            {
                best = time;
                splits = n;
            }
        }
        // About a workgroup a CU: eight waves read as much as several workgroups of
        // four, without parts to join. Below the given key tiles; one token each, us
        // split and so: 120 workgroups over 1000 keys, bf16 20.6, 18.1, four bits
        // 17.3, 14.2; over 8000 92, 104 and 37, 53; 160 over 2000 33.5, 29.5 and 22,
        // 20.5; over 8000 117, 114 and 47, 53; 240 over 2000 44, 40 and 26, 22; over
        // 8000 170, 167 and 59, 56; 100 over 1000 18.6, 17.7 and 15.8, 13.5, over 4000
        // 39, 43 and 24, 29.
        const long long most = blocks < 80 || blocks > 256 ? 0
                               : blocks < 112              ? 45
                               : blocks < 144              ? (p.four ? 50 : 150)
                               : blocks < 224              ? (p.four ? 100 : 256)
                                                           : 256;
        p.wide = splits > 1 && count <= most;
        p.one = p.more = parts(p.wide ? 1 : splits);
        return;
    }
    // (Without a window the rows of a chunk see, on the average, all but half of it.)
    const double average =
        p.mask.window > 0 ? count : std::max(1.0, (keys - 0.5 * std::min<long long>(c.max_rows, keys)) / kKeyTile);
    const TileTimes times(p, rows);
    if (p.tiles == 1)
    {
        const Split split = tile_splits(times, static_cast<long long>(c.heads) * c.sequences, average);
        p.one = p.more = parts(std::max(least, split.n));
        p.parts = p.one.splits;
        return;
    }
    // (A sequence's last row tile may have one row.)
    const long long most = std::min(static_cast<long long>(p.tiles) * c.sequences,
                                    static_cast<long long>(c.total_rows) * group / kTileRows + c.sequences);
    const Split split = tile_splits(times, c.heads * most, average);
    p.more = parts(split.n);
    // Where all row tiles see about as many keys, the last ones alone may be split.
    const long long fewest = std::max(1ll, std::min(keys, max_length - static_cast<long long>(c.max_rows)));
    if (split.n == 1 && 2 * fewest > keys)
    {
        const FirstSplit first = first_splits(times, c.heads * most, static_cast<long long>(c.heads) * c.sequences,
                                              p.tiles, average, split.time);
        if (first.n > 1)
        {
            const long long tokens = (static_cast<long long>(first.tiles) * kTileRows + group - 1) / group;
            p.more = parts(first.n);
            p.more.tiles = first.tiles;
            // (Of the last of them.)
            const long long last = std::min(count, ((fewest + tokens) >> kKeyShift) + 2);
            p.more.part_tiles = static_cast<int>((last + first.n - 1) / first.n);
            if (tokens * c.sequences < c.total_rows)
            {
                p.more.seq_rows = static_cast<int>(tokens);
                p.more.rows = tokens * c.sequences;
            }
        }
    }
    p.one = parts(1);
    // Single tokens and short chunks beside longer ones, if there can be any, are
    // dealt out by themselves; how many there are, and how long, is not known here,
    // so either kind is split only if few workgroups are there for it.
    const int one_rows = kTileRows / group;
    if (one_rows > 0 && c.total_rows - (c.sequences - 1ll) * c.max_rows <= one_rows)
    {
        const auto few = [&](long long blocks) {
            return blocks < 192 ? std::min((511 + blocks) / blocks, count / 8) : 1;
        };
        p.more = parts(few(c.heads * most));
        p.one = parts(std::max(least, few(c.heads * (c.sequences - 1ll))));
        if (static_cast<long long>(one_rows) * c.sequences < c.total_rows)
        {
            p.one.seq_rows = one_rows;
            p.one.rows = static_cast<long long>(one_rows) * c.sequences;
        }
    }
    // A workgroup without work takes about 0.8 ns of the launch, the list 4 us: a
    // chunk of 4096 rows beside 127 single tokens over 300 keys, 32/8 heads: 308
    // us, listed 185; beside 511: 916 and 306; beside 7: 183 and 174.
    const long long each = std::max(p.tiles - p.more.tiles + static_cast<long long>(p.more.tiles) * p.more.splits,
                                    static_cast<long long>(p.one.splits));
    const long long listed = static_cast<long long>(c.total_rows) * group / kTileRows * p.more.splits +
                             static_cast<long long>(c.sequences) * std::max(p.one.splits, p.more.splits);
    p.listed = (each * c.sequences - listed) * c.heads > 10000;
    p.parts = p.listed ? listed : each;
}

namespace
{

TileDeal tile_deal(const KvAttentionLaunch& p)
{
    return tile_deal(p.cache.heads * (p.listed ? 1 : p.cache.sequences), static_cast<int>(p.parts));
}

// The join of a sequence's rows: whether a wave takes one of them, for few rows
// and for many parts, and its workgroups, for many sequences no more than a
// single token needs.
struct MergeDeal
{
    bool one_row;
    int blocks;
};

MergeDeal merge_deal(const KvAttentionLaunch& p)
{
    const long long first = (static_cast<long long>(p.more.tiles) * kTileRows + p.group.d - 1) / p.group.d;
    const long long tokens = std::min(static_cast<long long>(p.cache.max_rows),
                                      p.more.splits > 1 ? first : kTileRows / p.group.d);
    MergeDeal d;
    d.one_row = tokens * p.heads.d * p.cache.sequences < 8192 ||
                std::max(p.one.splits, p.more.splits) > 16;
    const int each = d.one_row ? 4 : 16; // rows of a workgroup
    d.blocks = static_cast<int>(std::min((tokens * p.heads.d + each - 1) / each,
                                         std::max((p.heads.d + each - 1ll) / each, 8192ll / p.cache.sequences)));
    return d;
}

size_t partial_floats(const KvAttentionLaunch& p, const KvParts& k)
{
    return k.splits == 1 ? 0 : static_cast<size_t>(k.rows) * p.heads.d * k.splits * (p.head_dim + 2);
}

size_t list_bytes(const KvAttentionLaunch& p)
{
    return p.listed ? (2 * (p.cache.sequences + 1) * sizeof(int) + 15) / 16 * 16 : 0;
}

} // namespace

size_t kv_attention_workspace_bytes(const KvAttentionLaunch& p)
{
    return list_bytes(p) +
           (partial_floats(p, p.one) + (p.tiles > 1 && !p.few ? partial_floats(p, p.more) : 0)) * sizeof(float);
}

void kv_attention_set_workspace(KvAttentionLaunch& p, void* workspace)
{
    p.list = static_cast<int*>(workspace);
    p.one.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + list_bytes(p));
    p.more.partial = p.one.partial + (p.tiles > 1 && !p.few ? partial_floats(p, p.one) : 0);
}

bool kv_attention_fits(const KvAttentionLaunch& p)
{
    const long long most = 1ll << 23; // workgroups of a launch: their threads are counted in 32 bits
    if (p.heads.d / 4 >= most || static_cast<long long>(p.cache.heads) * p.cache.sequences >= most)
        return false;
    if (p.few)
        return static_cast<long long>(p.tiles) * p.cache.heads < most;
    if (p.parts >= most)
        return false;
    const TileDeal t = tile_deal(p);
    return 8ll * t.period * t.periods < most;
}

namespace
{

template <int D, bool F32, bool FOUR>
hipError_t launch(const KvAttentionLaunch& p, hipStream_t stream)
{
    if (p.few)
    {
        const dim3 grid(p.tiles * p.cache.heads, p.cache.sequences, p.one.splits);
        if (p.wide)
            hipLaunchKernelGGL((kv_rows_kernel<D, F32, FOUR, kWideWaves>), grid, dim3(kWideWaves * 64), 0, stream, p);
        else
            hipLaunchKernelGGL((kv_rows_kernel<D, F32, FOUR, kWaves>), grid, dim3(kWaves * 64), 0, stream, p);
    }
    else
    {
        if (p.listed)
        {
            hipLaunchKernelGGL(kv_list_kernel, dim3(1), dim3(kListThreads), 0, stream, p);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess)
                return e;
        }
        const TileDeal t = tile_deal(p);
        hipLaunchKernelGGL((kv_tile_kernel<D, F32, FOUR>), dim3(8u * t.period * t.periods), dim3(256), 0, stream, p, t);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (p.one.splits == 1 && p.more.splits == 1))
        return e;
    const MergeDeal m = merge_deal(p);
    const dim3 grid(m.blocks, p.cache.sequences);
    if (m.one_row)
        hipLaunchKernelGGL((kv_merge_kernel<D, F32, 4>), grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((kv_merge_kernel<D, F32, 1>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

} // namespace

hipError_t launch_kv_attention(const KvAttentionLaunch& p, hipStream_t stream)
{
    if (p.head_dim == 128)
        return p.four ? (p.f32 ? launch<128, true, true>(p, stream) : launch<128, false, true>(p, stream))
                      : (p.f32 ? launch<128, true, false>(p, stream) : launch<128, false, false>(p, stream));
    return p.four ? (p.f32 ? launch<64, true, true>(p, stream) : launch<64, false, true>(p, stream))
                  : (p.f32 ? launch<64, true, false>(p, stream) : launch<64, false, false>(p, stream));
}

} // namespace awa
