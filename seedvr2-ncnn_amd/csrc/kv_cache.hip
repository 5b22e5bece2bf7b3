// Rows into the pages of a key/value cache and out of them (gfx950).
//
// kv_append_kernel rotates new queries and keys, stores the keys and values at
// their slots and the queries where the attention reads them. Bound by memory:
// a row is read once and written once. A workgroup takes the rows of a few
// tokens; the (cos, sin) of a token's pairs are computed once and shared by its
// heads.
//
// Angles: positions of a long session are far from zero, so an angle's turns
// are a 64-bit fraction times the position, of which the whole turns fall off
// by overflow; the rest is within [-1/8, 1/8] turn of a quarter and goes
// through the Taylor series of sine and cosine in 64 bits. The rotation is in
// 64 bits too: a value next to a border of the 4-bit codes then falls where it
// does in exact arithmetic.
//
// 4-bit rows: 32 features share a power of two 2^e, the least with max |x| <=
// 7 * 2^e, so that no value is clipped by more than the half step that rounds
// it anyway; the codes are the hardware's e2m1 (nearest, ties to even) of x /
// 2^e. A group with a NaN or an infinity stands for NaN (byte 255).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "awa_device.h"
#include "kv_device.h"
#include "kv_kernels.h"

namespace awa
{
namespace
{

using namespace dev;

constexpr int kThreads = 256;
constexpr unsigned kInf = 0x7f800000u;

// (cos, sin) of a fraction of a turn: its nearest quarter, and the Taylor
// series of what is left (|x| <= pi / 4: terms behind x^17 are below 1e-18).
__device__ __forceinline__ double2 cos_sin_turns(unsigned long long turns)
{
    const unsigned quarter = static_cast<unsigned>((turns + (1ull << 61)) >> 62);
    const long long rest = static_cast<long long>(turns - (static_cast<unsigned long long>(quarter) << 62));
    const double x = static_cast<double>(rest) * (6.283185307179586476925 / 18446744073709551616.0);
    const double y = x * x;
    double s = 1.0 / 355687428096000.0;
    s = fma(s, y, -1.0 / 1307674368000.0);
    s = fma(s, y, 1.0 / 6227020800.0);
    s = fma(s, y, -1.0 / 39916800.0);
    s = fma(s, y, 1.0 / 362880.0);
    s = fma(s, y, -1.0 / 5040.0);
    s = fma(s, y, 1.0 / 120.0);
    s = fma(s, y, -1.0 / 6.0);
    s = fma(s * y, x, x);
    double c = 1.0 / 20922789888000.0;
    c = fma(c, y, -1.0 / 87178291200.0);
    c = fma(c, y, 1.0 / 479001600.0);
    c = fma(c, y, -1.0 / 3628800.0);
    c = fma(c, y, 1.0 / 40320.0);
    c = fma(c, y, -1.0 / 720.0);
    c = fma(c, y, 1.0 / 24.0);
    c = fma(c, y, -0.5);
    c = fma(c, y, 1.0);
    const double a = quarter & 1 ? s : c;
    const double b = quarter & 1 ? c : s;
    return make_double2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// x in fp32 rounded to odd: truncated, with the last bit set if anything was
// cut off. Rounding that to fewer bits is rounding x itself.
__device__ __forceinline__ float round_odd(double x)
{
    const float f = static_cast<float>(x);
    const double back = static_cast<double>(f);
    unsigned b = __float_as_uint(f);
    // An infinity that x overflowed to is the type's largest number again.
    if (back != x && !(b & 1u) && x == x)
        b += fabs(back) < fabs(x) ? 1u : -1u;
    return __uint_as_float(b);
}

// Sequence of packed row t, by the whole wave: the first that has it
// (sequences: none).
__device__ __forceinline__ int find_sequence(const KvView& c, int t)
{
    if (!c.cu)
        return t / c.max_rows;
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < c.sequences; i += 64)
    {
        const bool in = i + lane < c.sequences && c.cu[i + lane] <= t && t < c.cu[i + lane + 1];
        const unsigned long long found = __ballot(in);
        if (found)
            return i + __ffsll(found) - 1;
    }
    return c.sequences;
}

// Tells what does not fit together; one workgroup of a launch does it for all
// sequences, also those without rows.
__device__ __forceinline__ void tell_status(const KvView& c)
{
    if (!c.status || blockIdx.x != 0 || blockIdx.y != 0)
        return;
    unsigned bad = 0;
    for (int s = threadIdx.x; s < c.sequences; s += kThreads)
        bad |= kv_sequence(c, s).bad;
    if (bad)
        atomicOr(c.status, static_cast<int>(bad));
}

// Where a new row goes: slot < 0: nowhere (rows behind the last sequence, or
// of one that does not fit together). page < 0: its page is none of the pool's.
struct Place
{
    int slot, page;
};

__device__ __forceinline__ Place place_row(const KvView& c, int t)
{
    Place p{-1, -1};
    const int s = find_sequence(c, t);
    if (s >= c.sequences)
        return p;
    const KvSequence q = kv_sequence(c, s);
    const int j = t - q.first;
    if (j >= 0 && j < q.rows)
    {
        p.slot = q.length - q.rows + j;
        const int page = c.table[static_cast<long long>(s) * c.table_stride + (p.slot >> c.page_shift)];
        if (static_cast<unsigned>(page) < static_cast<unsigned>(c.pages))
            p.page = page;
        else if (c.status && (threadIdx.x & 63) == 0)
            atomicOr(c.status, AWA_KV_BAD_PAGE);
    }
    return p;
}

// Index of a row in its pool.
__device__ __forceinline__ size_t pool_row(const KvView& c, const Place& p, int head)
{
    return ((static_cast<size_t>(p.page) * c.heads + head) << c.page_shift) + (p.slot & ((1 << c.page_shift) - 1));
}

template <bool F32>
__device__ __forceinline__ void load8(const unsigned char* p, float (&v)[8])
{
    if (F32)
    {
        const float4 a = *reinterpret_cast<const float4*>(p);
        const float4 b = *reinterpret_cast<const float4*>(p + 16);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    else
    {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
        v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
    }
}

template <bool F32>
__device__ __forceinline__ void store8(unsigned char* p, const float (&v)[8])
{
    if (F32)
    {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 16) = make_float4(v[4], v[5], v[6], v[7]);
    }
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]),
                                                  cvt_pk_bf16(v[4], v[5]), cvt_pk_bf16(v[6], v[7]));
}

// Eight features of a row in four bits: the codes in one word; the four lanes
// of a group share the scale byte, which the first of them stores.
__device__ __forceinline__ void store8_four(unsigned char* codes, unsigned char* scale, bool first,
                                            const float (&v)[8])
{
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++)
        top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, false)));
    top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xF, 0xF, false)));
    // 7 * 2^e = 1.75 * 2^(e + 2).
    int byte = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u);
    byte = max(byte, 1);
    unsigned word = 0;
    if (top < kInf)
    {
        const float unit = __uint_as_float(static_cast<unsigned>(byte) << 23);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], unit, 0);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], unit, 1);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], unit, 2);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], unit, 3);
    }
    else
        byte = 255;
    *reinterpret_cast<unsigned*>(codes) = word;
    if (first)
        *scale = static_cast<unsigned char>(byte);
}

// TOKENS tokens a workgroup and blockIdx.y's part of their heads; LANES lanes
// hold a row, eight features each.
template <bool F32, bool FOUR, int D, int TOKENS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvAppendLaunch p, int heads_part)
{
    constexpr int kLanes = D / 8;
    constexpr int kSlots = kThreads / kLanes; // rows at a time
    constexpr int kElem = F32 ? 4 : 2;
    __shared__ double2 turn[TOKENS][kRopeMaxPairs];
    __shared__ Place places[TOKENS];
    const int tid = threadIdx.x;
    const int wave = tid >> 6;
    const int t0 = blockIdx.x * TOKENS;
    const KvView& c = p.cache;

    for (int i = wave; i < TOKENS; i += kThreads / 64)
    {
        const Place at = t0 + i < c.total_rows ? place_row(c, t0 + i) : Place{-1, -1};
        if ((tid & 63) == 0)
            places[i] = at;
        if (p.rope.axes > 0 && at.slot >= 0)
        {
            const int pair = tid & 63;
            if (pair < p.rope.pairs * p.rope.axes)
            {
                const int axis = pair / p.rope.pairs;
                const int x = p.positions ? p.positions[static_cast<long long>(t0 + i) * p.rope.axes + axis] : at.slot;
                turn[i][pair] = cos_sin_turns(static_cast<unsigned long long>(static_cast<long long>(x)) *
                                              p.rope.turns[pair - axis * p.rope.pairs]);
            }
        }
    }
    __syncthreads();
    tell_status(c);

    const int l = tid % kLanes;
    const int heads = (p.q.data ? p.q_heads : 0) + 2 * c.heads;
    const int head0 = blockIdx.y * heads_part;
    const int part = min(heads_part, heads - head0);
    const int pairs = p.rope.pairs * p.rope.axes;
    for (int i = tid / kLanes; i < TOKENS * part; i += kSlots)
    {
        const int token = i / part;
        int head = head0 + i - token * part;
        const Place at = places[token];
        if (at.slot < 0)
            continue;
        // Queries first, then keys, then values.
        const int q_heads = heads - 2 * c.heads;
        const int kind = head < q_heads ? 0 : head < q_heads + c.heads ? 1 : 2;
        head -= kind == 0 ? 0 : kind == 1 ? q_heads : q_heads + c.heads;
        const KvRowsSource& src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
        const long long t = t0 + token;
        float v[8];
        load8<F32>(src.data + t * src.stride + (static_cast<long long>(head) * D + 8 * l) * kElem, v);
        if (kind < 2 && p.rope.axes > 0)
        {
            float other[8];
            int step = 0;
            bool second = false;
            if (p.rope.halves)
            {
                // The other feature of each pair is `step` lanes away.
                step = pairs / 8;
                second = l >= step;
                const int from = l < 2 * step ? (second ? l - step : l + step) : l;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    other[e] = __shfl(v[e], from, kLanes);
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const int f = 8 * l + e;
                const int pair = p.rope.halves ? f - (second ? pairs : 0) : f >> 1;
                const bool odd = p.rope.halves ? second : (e & 1) != 0;
                if (f < 2 * pairs)
                {
                    const double2 cs = turn[token][pair];
                    const double a = v[e];
                    if (!p.rope.halves && !(e & 1))
                        other[e + 1] = v[e], other[e] = v[e + 1];
                    const double b = other[e];
                    const double r = fma(a, cs.x, odd ? b * cs.y : -(b * cs.y));
                    v[e] = F32 && kind == 0 ? static_cast<float>(r) : round_odd(r);
                }
            }
        }
        if (kind == 0)
        {
            store8<F32>(const_cast<unsigned char*>(p.q_out.data) + t * p.q_out.stride +
                            (static_cast<long long>(head) * D + 8 * l) * kElem,
                        v);
            continue;
        }
        if (at.page < 0)
            continue;
        const size_t row = pool_row(c, at, head);
        unsigned char* const pool = kind == 1 ? c.k : c.v;
        if (FOUR)
            store8_four(pool + row * (D / 2) + 4 * l, (kind == 1 ? c.k_scale : c.v_scale) + row * (D / kKvGroup) + l / 4,
                        l % 4 == 0, v);
        else
            store8<false>(pool + (row * D + 8 * l) * 2, v);
    }
}

// The other way: the rows that the cache holds at the new rows' slots. Rows
// whose page is none of the pool's are left as they were.
template <bool F32, bool FOUR, int D, int TOKENS>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const KvReadLaunch p, int heads_part)
{
    constexpr int kLanes = D / 8;
    constexpr int kSlots = kThreads / kLanes;
    constexpr int kElem = F32 ? 4 : 2;
    __shared__ Place places[TOKENS];
    const int tid = threadIdx.x;
    const int t0 = blockIdx.x * TOKENS;
    const KvView& c = p.cache;
    for (int i = tid >> 6; i < TOKENS; i += kThreads / 64)
    {
        const Place at = t0 + i < c.total_rows ? place_row(c, t0 + i) : Place{-1, -1};
        if ((tid & 63) == 0)
            places[i] = at;
    }
    __syncthreads();
    tell_status(c);
    const int l = tid % kLanes;
    const int heads = 2 * c.heads;
    const int head0 = blockIdx.y * heads_part;
    const int part = min(heads_part, heads - head0);
    for (int i = tid / kLanes; i < TOKENS * part; i += kSlots)
    {
        const int token = i / part;
        int head = head0 + i - token * part;
        const Place at = places[token];
        if (at.slot < 0 || at.page < 0)
            continue;
        const bool key = head < c.heads;
        head -= key ? 0 : c.heads;
        const size_t row = pool_row(c, at, head);
        const unsigned char* const pool = key ? c.k : c.v;
        float v[8];
        if (FOUR)
        {
            const unsigned word = *reinterpret_cast<const unsigned*>(pool + row * (D / 2) + 4 * l);
            const unsigned byte = (key ? c.k_scale : c.v_scale)[row * (D / kKvGroup) + l / 4];
            const float unit = four_unit(byte);
            four_values(word, unit, v);
        }
        else
            load8<false>(pool + (row * D + 8 * l) * 2, v);
        const KvRowsSource& to = key ? p.k : p.v;
        store8<F32>(const_cast<unsigned char*>(to.data) + (static_cast<long long>(t0) + token) * to.stride +
                        (static_cast<long long>(head) * D + 8 * l) * kElem,
                    v);
    }
}

// Tokens a workgroup and heads a part: whole tokens, four at a time, where
// they fill the device, else a row a lane group.
struct Deal
{
    bool four_tokens;
    int heads_part;
    dim3 grid;
};

Deal deal(int total, int heads, int head_dim)
{
    Deal d;
    d.four_tokens = total >= 2048;
    d.heads_part = d.four_tokens ? heads : kThreads / (head_dim / 8);
    d.grid = dim3(d.four_tokens ? (total + 3) / 4 : total, (heads + d.heads_part - 1) / d.heads_part);
    return d;
}

template <bool F32, bool FOUR, int D>
void append_to(const KvAppendLaunch& p, const Deal& d, hipStream_t stream)
{
    if (d.four_tokens)
        hipLaunchKernelGGL((kv_append_kernel<F32, FOUR, D, 4>), d.grid, dim3(kThreads), 0, stream, p, d.heads_part);
    else
        hipLaunchKernelGGL((kv_append_kernel<F32, FOUR, D, 1>), d.grid, dim3(kThreads), 0, stream, p, d.heads_part);
}

template <bool F32, bool FOUR, int D>
void read_from(const KvReadLaunch& p, const Deal& d, hipStream_t stream)
{
    if (d.four_tokens)
        hipLaunchKernelGGL((kv_read_kernel<F32, FOUR, D, 4>), d.grid, dim3(kThreads), 0, stream, p, d.heads_part);
    else
        hipLaunchKernelGGL((kv_read_kernel<F32, FOUR, D, 1>), d.grid, dim3(kThreads), 0, stream, p, d.heads_part);
}

} // namespace

hipError_t launch_kv_append(const KvAppendLaunch& p, hipStream_t stream)
{
    const Deal d = deal(p.cache.total_rows, (p.q.data ? p.q_heads : 0) + 2 * p.cache.heads, p.head_dim);
    if (p.head_dim == 128)
        p.four ? (p.f32 ? append_to<true, true, 128>(p, d, stream) : append_to<false, true, 128>(p, d, stream))
               : (p.f32 ? append_to<true, false, 128>(p, d, stream) : append_to<false, false, 128>(p, d, stream));
    else
        p.four ? (p.f32 ? append_to<true, true, 64>(p, d, stream) : append_to<false, true, 64>(p, d, stream))
               : (p.f32 ? append_to<true, false, 64>(p, d, stream) : append_to<false, false, 64>(p, d, stream));
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvReadLaunch& p, hipStream_t stream)
{
    const Deal d = deal(p.cache.total_rows, 2 * p.cache.heads, p.head_dim);
    if (p.head_dim == 128)
        p.four ? (p.f32 ? read_from<true, true, 128>(p, d, stream) : read_from<false, true, 128>(p, d, stream))
               : (p.f32 ? read_from<true, false, 128>(p, d, stream) : read_from<false, false, 128>(p, d, stream));
    else
        p.four ? (p.f32 ? read_from<true, true, 64>(p, d, stream) : read_from<false, true, 64>(p, d, stream))
               : (p.f32 ? read_from<true, false, 64>(p, d, stream) : read_from<false, false, 64>(p, d, stream));
    return hipGetLastError();
}

} // namespace awa
