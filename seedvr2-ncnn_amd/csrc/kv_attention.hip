// Attention of new rows over a key/value cache in pages (gfx950): a sliding
// window and first tokens that stay visible, pages in bf16 or in four bits.
//
// out = sum_k exp(scale q.k - m) v_k / sum_k exp(scale q.k - m) over the keys
// a row sees, in one pass with the running maximum m. The rows of one sequence
// that share a key/value head (its new tokens times the query heads of a
// group) are packed into row tiles; the key tiles that a row tile sees (those
// of the sinks, then those of the window) are dealt to `splits` workgroups,
// whose parts kv_merge_kernel joins.
//
// fp32 rows: queries and probabilities are three bf16 pieces (all 24 bits), so
// that products with the cache's values are exact and sums are fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

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

constexpr int kRowTile = 16; // rows of kv_rows_kernel's tile
constexpr int kKeyTile = 32;
constexpr int kKeyShift = 5;
constexpr int kWaves = 4;

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

// One row tile of 16 rows, one part of its keys: each of the four waves takes
// every fourth key tile (32 keys) by itself, with K from memory straight into
// the MFMA operand registers and V through the wave's own LDS, from which it
// is read transposed; the waves' results are joined at the end. Bound by
// reading the cache.
//
// S^T = K Q^T (16x16x32): lane (r = lane % 16, g = lane / 16) holds row r's
// scores of keys 4 g + [0, 4) of each 16. Those of two blocks are, in that
// order, the eight values a lane holds of the PV product's operand P^T; V^T is
// read in the same key order.
template <int D, bool F32, bool FOUR>
__global__ __launch_bounds__(kWaves * 64) void kv_rows_kernel(const KvAttentionLaunch p, int row_tiles)
{
    constexpr int kPieces = F32 ? 3 : 1;
    constexpr int kChunks = D / 32;
    constexpr int kBlocks = D / 16;
    constexpr int kPitch = D + 32; // V rows in LDS, elements
    constexpr int kElem = F32 ? 4 : 2;
    constexpr int kVBytes = kKeyTile * kPitch * 2;
    constexpr int kOBytes = kRowTile * D * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[kWaves][kVBytes > kOBytes ? kVBytes : kOBytes];
    __shared__ float stats[kWaves][kRowTile][2];

    const KvView& c = p.cache;
    const int seq = blockIdx.y;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15;
    const int g = lane >> 4;
    int block = blockIdx.x;
    const int split = block % p.splits;
    block /= p.splits;
    const int tile = block % row_tiles;
    const int head = block / row_tiles;

    const KvSequence s = kv_sequence(c, seq);
    if (s.bad && c.status && threadIdx.x == 0)
        atomicOr(c.status, static_cast<int>(s.bad));
    const int rows = s.rows * p.group;
    const int row0 = tile * kRowTile;
    if (row0 >= rows)
        return;
    const int last = min(row0 + kRowTile, rows) - 1;
    const int slot0 = s.length - s.rows;
    const KvSpan span_first = kv_span(p.mask, slot0 + row0 / p.group, s.length);
    const KvSpan span_last = kv_span(p.mask, slot0 + last / p.group, s.length);

    // This lane's row (rows past the end repeat the last; they are not stored).
    const int row = min(row0 + r, last);
    const int token = row / p.group;
    const int q_head = head * p.group + row - token * p.group;
    const KvSpan span = kv_span(p.mask, slot0 + token, s.length);
    bf16x8 q[kChunks][kPieces];
    {
        const unsigned char* src =
            p.q.data + static_cast<long long>(s.first + token) * p.q.stride + static_cast<long long>(q_head) * D * kElem;
#pragma unroll
        for (int i = 0; i < kChunks; i++)
        {
            const int feature = 32 * i + 8 * g;
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

    const KvTiles tiles = kv_tiles(span_first, span_last, kKeyShift);
    const int count = tiles.sinks + tiles.rest;
    const int part_end = kv_part(count, split + 1, p.splits);

    f32x4 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    float row_max = -INFINITY;
    float row_sum = 0.f;
    unsigned bad = 0;

    const int* const table = c.table + static_cast<long long>(seq) * c.table_stride;
    const int slot_mask = (1 << c.page_shift) - 1;
    unsigned char* const v_lds = lds[wave];

    for (int i = kv_part(count, split, p.splits) + wave; i < part_end; i += kWaves)
    {
        const int key0 = (i < tiles.sinks ? i : tiles.begin + i - tiles.sinks) << kKeyShift;
        // Pages of the two blocks of 16 keys (a page holds whole blocks).
        size_t base[2];
        bool there[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
        {
            const int key = key0 + 16 * b;
            const bool in = key < span_last.end;
            const int page = table[(in ? key : key0) >> c.page_shift];
            const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(c.pages);
            there[b] = in && ok;
            if (!ok)
                bad = AWA_KV_BAD_PAGE;
            base[b] = (((ok ? static_cast<size_t>(page) : 0) * c.heads + head) << c.page_shift) + (key & slot_mask);
        }

        // K rows: lane r of block b holds key 16 b + r.
        bf16x8 k[2][kChunks];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int j = 0; j < kChunks; j++)
            {
                const size_t at = base[b] + r;
                if (FOUR)
                {
                    const unsigned w = *reinterpret_cast<const unsigned*>(c.k + at * (D / 2) + 16 * j + 4 * g);
                    const float unit = four_unit(c.k_scale[at * (D / kKvGroup) + j]);
                    float v[8];
                    four_values(w, unit, v);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        k[b][j][e] = static_cast<__bf16>(v[e]);
                }
                else
                    k[b][j] = *reinterpret_cast<const bf16x8*>(c.k + (at * D + 32 * j + 8 * g) * 2);
            }

        // V rows into LDS; keys that no row of the tile sees as zeros.
        constexpr int kRowLanes = D / 8;
        constexpr int kRowsPass = 64 / kRowLanes;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < kKeyTile / kRowsPass; j++)
        {
            const int local = j * kRowsPass + lane / kRowLanes;
            const int chunk = lane % kRowLanes;
            const int key = key0 + local;
            const int b = local >> 4;
            const size_t at = (b ? base[1] : base[0]) + (local & 15);
            const bool seen = (b ? there[1] : there[0]) && key < span_last.end &&
                              (key >= span_first.begin || key < span_last.sinks);
            uint4 w;
            if (FOUR)
            {
                const unsigned codes = *reinterpret_cast<const unsigned*>(c.v + at * (D / 2) + 4 * chunk);
                const float unit = four_unit(c.v_scale[at * (D / kKvGroup) + chunk / 4]);
                float v[8];
                four_values(codes, unit, v);
                w = make_uint4(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]), cvt_pk_bf16(v[4], v[5]),
                               cvt_pk_bf16(v[6], v[7]));
            }
            else
                w = *reinterpret_cast<const uint4*>(c.v + (at * D + 8 * chunk) * 2);
            if (!seen)
                w = make_uint4(0, 0, 0, 0);
            const unsigned words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                finite = finite && (words[e] & 0x7f80u) != 0x7f80u && (words[e] & 0x7f800000u) != 0x7f800000u;
            *reinterpret_cast<uint4*>(v_lds + (local * kPitch + 8 * chunk) * 2) = w;
        }

        f32x4 acc[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
        {
            acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < kChunks; j++)
#pragma unroll
                for (int e = kPieces - 1; e >= 0; e--)
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[b][j], q[j][e], acc[b], 0, 0, 0);
        }

        float x[8];
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++)
        {
            const int key = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
            const bool seen = there[e >> 2] && key < span.end && (key >= span.begin || key < span.sinks);
            x[e] = seen ? acc[e >> 2][e & 3] * p.scale_log2 : -INFINITY;
            top = fmaxf(top, x[e]);
        }
        top = max_xor32(max_xor16(top));
        if (__any(top > row_max))
        {
            const float next = fmaxf(row_max, top);
            const float alpha = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(row_max - next);
            row_max = next;
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

        // The wave's LDS writes before its transposed reads.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (__all(finite))
        {
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
        }
        else
        {
            // A NaN or an infinity among the values: a product with the zero
            // weight of a row that does not see it would be NaN, so those rows
            // are left out key by key.
#pragma unroll 1
            for (int key = 0; key < kKeyTile; key++)
            {
                const int owner = (key & 15) >> 2;
                float weight = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    weight = e == (key >> 4) * 4 + (key & 3) ? (F32 ? x[e] : static_cast<float>(w[0][e])) : weight;
                weight = __shfl(weight, owner * 16 + r, 64);
                const int k_at = key0 + key;
                const bool seen =
                    there[key >> 4] && k_at < span.end && (k_at >= span.begin || k_at < span.sinks);
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                    {
                        const uint16_t bits =
                            *reinterpret_cast<const uint16_t*>(v_lds + (key * kPitch + 16 * b + 4 * g + e) * 2);
                        const float value = __uint_as_float(static_cast<unsigned>(bits) << 16);
                        if (seen)
                            o[b][e] = fmaf(weight, value, o[b][e]);
                    }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (bad && c.status && lane == 0)
        atomicOr(c.status, static_cast<int>(bad));

    // Join the waves: each lane group holds a part of its row's sum.
    row_sum = sum_xor32(sum_xor16(row_sum));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
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
    constexpr int kPer = kRowTile * D / (kWaves * 64); // features a thread
    const int out_row = threadIdx.x * kPer / D;
    const int f0 = threadIdx.x * kPer % D;
    if (row0 + out_row > last)
        return;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; i++)
        m = fmaxf(m, stats[i][out_row][0]);
    const float from = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    float v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++)
        v[e] = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; i++)
    {
        const float weight = __builtin_amdgcn_exp2f(stats[i][out_row][0] - from);
        sum += weight * stats[i][out_row][1];
        const float* const part = reinterpret_cast<const float*>(lds[i]) + out_row * D + f0;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            v[e] = fmaf(weight, part[e], v[e]);
    }
    const int out_token = (row0 + out_row) / p.group;
    const int out_head = head * p.group + (row0 + out_row) - out_token * p.group;
    const long long t = s.first + out_token;
    if (p.splits > 1)
    {
        const size_t heads = static_cast<size_t>(c.heads) * p.group;
        const size_t all = static_cast<size_t>(c.total_rows) * heads;
        const size_t at = split * all + t * heads + out_head;
        float* const dst = p.partial + at * D + f0;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            dst[e] = v[e];
        if (f0 == 0)
        {
            float* const st = p.partial + p.splits * all * D + at * 2;
            st[0] = m;
            st[1] = sum;
        }
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    unsigned char* const dst = const_cast<unsigned char*>(p.out.data) + t * p.out.stride +
                               (static_cast<long long>(out_head) * D + f0) * kElem;
#pragma unroll
    for (int e = 0; e < kPer; e += 4)
    {
        if (F32)
            store4(reinterpret_cast<float*>(dst) + e, v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv);
        else
            store4(reinterpret_cast<uint16_t*>(dst) + e, v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv);
    }
}

// Joins the parts of a row: M = max m_i, out = sum 2^(m_i - M) o_i / sum
// 2^(m_i - M) l_i, in the parts' order. One wave a row and query head.
template <int D, bool F32>
__global__ __launch_bounds__(256) void kv_merge_kernel(const KvAttentionLaunch p)
{
    constexpr int kPer = D / 64;
    const KvView& c = p.cache;
    const KvSequence s = kv_sequence(c, blockIdx.y);
    const int heads = c.heads * p.group;
    const long long i = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (i >= static_cast<long long>(s.rows) * heads)
        return;
    const int lane = threadIdx.x & 63;
    const size_t all = static_cast<size_t>(c.total_rows) * heads;
    const size_t at = static_cast<size_t>(s.first) * heads + i;
    const float* const stats = p.partial + p.splits * all * D;
    float m = -INFINITY;
    for (int j = 0; j < p.splits; j++)
        m = fmaxf(m, stats[(j * all + at) * 2]);
    const float from = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    float v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++)
        v[e] = 0.f;
    for (int j = 0; j < p.splits; j++)
    {
        const float weight = __builtin_amdgcn_exp2f(stats[(j * all + at) * 2] - from);
        sum += weight * stats[(j * all + at) * 2 + 1];
        const float* const part = p.partial + (j * all + at) * D + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            v[e] = fmaf(weight, part[e], v[e]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const long long token = i / heads;
    unsigned char* const dst = const_cast<unsigned char*>(p.out.data) + (s.first + token) * p.out.stride +
                               (i - token * heads) * D * (F32 ? 4 : 2);
#pragma unroll
    for (int e = 0; e < kPer; e++)
    {
        if (F32)
            reinterpret_cast<float*>(dst)[lane * kPer + e] = v[e] * inv;
        else
            reinterpret_cast<__bf16*>(dst)[lane * kPer + e] = static_cast<__bf16>(v[e] * inv);
    }
}

template <int D, bool F32, bool FOUR>
hipError_t launch(const KvAttentionLaunch& p, hipStream_t stream)
{
    const int row_tiles = (p.cache.max_rows * p.group + kRowTile - 1) / kRowTile;
    hipLaunchKernelGGL((kv_rows_kernel<D, F32, FOUR>), dim3(row_tiles * p.cache.heads * p.splits, p.cache.sequences),
                       dim3(kWaves * 64), 0, stream, p, row_tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1)
        return e;
    hipLaunchKernelGGL((kv_merge_kernel<D, F32>),
                       dim3((p.cache.max_rows * p.cache.heads * p.group + 3) / 4, p.cache.sequences), dim3(256), 0,
                       stream, p);
    return hipGetLastError();
}

} // namespace

int kv_attention_splits(const KvView& c, int group, const KvMaskRule& mask, int max_length)
{
    // Keys that a row tile may see, and the workgroups without splitting.
    long long keys = max_length;
    if (mask.window > 0)
        keys = std::min(keys, static_cast<long long>(mask.window) + mask.sinks + mask.block + c.max_rows);
    const long long tiles = (static_cast<long long>(c.max_rows) * group + kRowTile - 1) / kRowTile;
    const long long blocks = tiles * c.heads * c.sequences;
    const long long most = std::max(1ll, keys / 256);
    return static_cast<int>(std::min({most, std::max(1ll, 2048 / blocks), 64ll}));
}

size_t kv_attention_partial_bytes(const KvView& c, int group, int head_dim, int splits)
{
    return splits == 1 ? 0
                       : static_cast<size_t>(c.total_rows) * c.heads * group * splits * (head_dim + 2) * sizeof(float);
}

hipError_t launch_kv_attention(const KvAttentionLaunch& p, hipStream_t stream)
{
    if (p.head_dim == 128)
        return p.four ? (p.f32 ? launch<128, true, true>(p, stream) : launch<128, false, true>(p, stream))
                      : (p.f32 ? launch<128, true, false>(p, stream) : launch<128, false, false>(p, stream));
    return p.four ? (p.f32 ? launch<64, true, true>(p, stream) : launch<64, false, true>(p, stream))
                  : (p.f32 ? launch<64, true, false>(p, stream) : launch<64, false, false>(p, stream));
}

} // namespace awa
