// Rows into the pages of a key/value cache and out of them (gfx950).
//
// kv_append_kernel rotates new queries and keys, stores the keys and values at
// their slots and the queries where the attention reads them. Bound by memory:
// a row is read once and written once. A workgroup takes the rows of a few
// tokens; the (cos, sin) of a token's pairs are computed once and shared by its
// heads. 13311 tokens of 20 heads of 128, queries, keys and values in bf16: 85 us,
// 4.8 TB/s (a copy reaches 4.9); 16 tokens: 4.5 us, a launch.
//
// Angles: positions of a long session are far from zero, so an angle's turns
// are a 64-bit fraction times the position, of which the whole turns fall off
// by overflow; the rest is within [-1/8, 1/8] turn of a quarter and goes
// through the Taylor series of sine and cosine in 64 bits. Rows that stay fp32
// or become bf16 are rotated in fp32 with (cos, sin) rounded to fp32: off by at
// most 2^-24 (|a| + 2 |b| + |r|) for r = a cos - b sin, far below half a step of
// bf16. Keys that become four bits are rotated in 64 bits, and rounded once: a
// value next to a border of the codes, of which a step is a third of the value,
// then falls where it does in exact arithmetic.
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
    // (One with more rows than there may be takes no part.)
    const auto has = [&](int s) {
        const int from = c.cu[s], to = c.cu[s + 1];
        return from >= 0 && from <= t && t < to && to - from <= c.max_rows;
    };
    // The first that ends behind t, in 64ths of what is left; with cu_rows in
    // order it has t.
    if (c.sequences > 64)
    {
        int step = 1, s = 0;
        while (step * 64 < c.sequences)
            step *= 64;
        for (; step > 0; step /= 64)
        {
            const int at = s + (lane + 1) * step;
            const unsigned long long not_yet = __ballot(at <= c.sequences && c.cu[min(at, c.sequences)] <= t);
            s += (not_yet == ~0ull ? 64 : __ffsll(~not_yet) - 1) * step;
        }
        if (s < c.sequences && has(s))
            return s;
    }
    for (int i = 0; i < c.sequences; i += 64)
    {
        const bool in = i + lane < c.sequences && has(i + lane);
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

// Index of a row in its pool (of less than 2^31 rows).
__device__ __forceinline__ size_t pool_row(const KvView& c, const Place& p, int head)
{
    return static_cast<unsigned>(((p.page * c.heads + head) << c.page_shift) +
                                 (p.slot & ((1 << c.page_shift) - 1)));
}

// Eight features as they lie in memory.
template <bool F32>
struct Raw8
{
    uint4 a, b;
};

template <bool F32>
__device__ __forceinline__ Raw8<F32> load_raw(const unsigned char* p)
{
    Raw8<F32> r;
    r.a = *reinterpret_cast<const uint4*>(p);
    if (F32)
        r.b = *reinterpret_cast<const uint4*>(p + 16);
    return r;
}

template <bool F32>
__device__ __forceinline__ void values8(const Raw8<F32>& r, float (&v)[8])
{
    if (F32)
    {
        v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y), v[2] = __uint_as_float(r.a.z);
        v[3] = __uint_as_float(r.a.w), v[4] = __uint_as_float(r.b.x), v[5] = __uint_as_float(r.b.y);
        v[6] = __uint_as_float(r.b.z), v[7] = __uint_as_float(r.b.w);
    }
    else
    {
        v[0] = bf16_lo(r.a.x), v[1] = bf16_hi(r.a.x), v[2] = bf16_lo(r.a.y), v[3] = bf16_hi(r.a.y);
        v[4] = bf16_lo(r.a.z), v[5] = bf16_hi(r.a.z), v[6] = bf16_lo(r.a.w), v[7] = bf16_hi(r.a.w);
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

// How rows turn: not at all, neighbouring features, or the halves of a row.
enum
{
    kStill,
    kNeighbours,
    kHalves
};

// a cos + b sin.
__device__ __forceinline__ float turned(float a, float b, float c, float s)
{
    return fmaf(a, c, b * s);
}

__device__ __forceinline__ float turned(float a, float b, double c, double s)
{
    return round_odd(fma(static_cast<double>(a), c, static_cast<double>(b) * s));
}

// Eight features of a row, lane l of the row's; features behind the last pair
// stay.
template <int STYLE, int D, typename T2>
__device__ __forceinline__ void rotate8(float (&v)[8], int l, int pairs, const T2* turn)
{
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        x[e] = v[e];
    if (STYLE == kNeighbours)
    {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
        {
            const T2 cs = turn[4 * l + e / 2];
            v[e] = turned(x[e], x[e + 1], cs.x, -cs.y);
            v[e + 1] = turned(x[e + 1], x[e], cs.x, cs.y);
        }
    }
    else if (STYLE == kHalves)
    {
        // The other feature of each pair is `step` lanes away.
        const int step = pairs / 8;
        const bool second = l >= step;
        const int from = l < 2 * step ? (second ? l - step : l + step) : 0;
        const T2* const cs8 = turn + (l < 2 * step ? 8 * (second ? l - step : l) : 0);
#pragma unroll
        for (int e = 0; e < 8; e++)
        {
            const T2 cs = cs8[e];
            v[e] = turned(x[e], __shfl(x[e], from, D / 8), cs.x, second ? cs.y : -cs.y);
        }
    }
    if (STYLE && 2 * pairs < D)
    {
        const int left = 2 * pairs - 8 * l;
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = e < left ? v[e] : x[e];
    }
}

// TOKENS tokens a workgroup and blockIdx.y's part of their heads; LANES lanes
// hold a row, eight features each. Bound by memory and, next, by the steps that
// a row of 256 bytes takes (a quarter of a wave): queries, keys and values each
// have a loop of their own, without a choice in it.
template <bool F32, bool FOUR, int D, int TOKENS, int STYLE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvAppendLaunch p, int heads_part)
{
    constexpr int kLanes = D / 8;
    constexpr int kSlots = kThreads / kLanes; // rows at a time
    constexpr int kElem = F32 ? 4 : 2;
    __shared__ float2 turn[STYLE ? TOKENS : 1][kRopeMaxPairs];
    __shared__ double2 exact_turn[STYLE && FOUR ? TOKENS : 1][kRopeMaxPairs];
    __shared__ Place places[TOKENS];
    const int tid = threadIdx.x;
    const int t0 = blockIdx.x * TOKENS;
    const KvView& c = p.cache;
    const int pairs = p.rope.pairs * p.rope.axes;

    for (int i = tid >> 6; i < TOKENS; i += kThreads / 64)
    {
        const int lane = tid & 63;
        const Place at = t0 + i < c.total_rows ? place_row(c, t0 + i) : Place{-1, -1};
        if (lane == 0)
            places[i] = at;
        if (STYLE && at.slot >= 0 && lane < pairs)
        {
            const int axis = lane / p.rope.pairs;
            const int x = p.positions ? p.positions[static_cast<long long>(t0 + i) * p.rope.axes + axis] : at.slot;
            const double2 cs = cos_sin_turns(static_cast<unsigned long long>(static_cast<long long>(x)) *
                                             p.rope.turns[lane - axis * p.rope.pairs]);
            turn[i][lane] = make_float2(static_cast<float>(cs.x), static_cast<float>(cs.y));
            if (FOUR)
                exact_turn[i][lane] = cs;
        }
    }
    __syncthreads();
    tell_status(c);

    const int l = tid % kLanes;
    const int q_heads = p.q.data ? p.q_heads : 0;
    const int head0 = blockIdx.y * heads_part;
    // All rows of one kind, heads [first, first + count) of the launch's.
    auto each_row = [&](int first, int count, const KvRowsSource& src, auto row) {
        const int lo = max(head0 - first, 0);
        const int n = min(head0 + heads_part - first, count) - lo;
        if (n <= 0)
            return;
        int token = 0, head = lo + tid / kLanes;
        while (true)
        {
            while (head >= lo + n && token < TOKENS)
            {
                head -= n;
                token++;
            }
            if (token >= TOKENS)
                return;
            const Place at = places[token];
            if (at.slot >= 0)
            {
                float v[8];
                values8<F32>(load_raw<F32>(src.data + static_cast<long long>(t0 + token) * src.stride +
                                           (head * D + 8 * l) * kElem),
                             v);
                row(v, at, token, head);
            }
            head += kSlots;
        }
    };
    if (STYLE)
        each_row(0, q_heads, p.q, [&](float (&v)[8], const Place&, int token, int head) {
            rotate8<STYLE, D>(v, l, pairs, turn[token]);
            store8<F32>(const_cast<unsigned char*>(p.q_out.data) +
                            static_cast<long long>(t0 + token) * p.q_out.stride + (head * D + 8 * l) * kElem,
                        v);
        });
    each_row(q_heads, c.heads, p.k, [&](float (&v)[8], const Place& at, int token, int head) {
        if (FOUR)
            rotate8<STYLE, D>(v, l, pairs, exact_turn[token]);
        else
            rotate8<STYLE, D>(v, l, pairs, turn[token]);
        if (at.page < 0)
            return;
        const size_t r = pool_row(c, at, head);
        if (FOUR)
            store8_four(c.k + r * (D / 2) + 4 * l, c.k_scale + r * (D / kKvGroup) + l / 4, l % 4 == 0, v);
        else
            store8<false>(c.k + (r * D + 8 * l) * 2, v);
    });
    each_row(q_heads + c.heads, c.heads, p.v, [&](float (&v)[8], const Place& at, int, int head) {
        if (at.page < 0)
            return;
        const size_t r = pool_row(c, at, head);
        if (FOUR)
            store8_four(c.v + r * (D / 2) + 4 * l, c.v_scale + r * (D / kKvGroup) + l / 4, l % 4 == 0, v);
        else
            store8<false>(c.v + (r * D + 8 * l) * 2, v);
    });
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
            values8<false>(load_raw<false>(pool + (row * D + 8 * l) * 2), v);
        const KvRowsSource& to = key ? p.k : p.v;
        store8<F32>(const_cast<unsigned char*>(to.data) + (static_cast<long long>(t0) + token) * to.stride +
                        (static_cast<long long>(head) * D + 8 * l) * kElem,
                    v);
    }
}

// Tokens a workgroup and heads a part: whole tokens, four at a time, where
// they fill the device, else a row a lane group. 20 heads of 128, bf16 (us), one
// token and four: 512 tokens 9.6, 11; 1024 10, 13; 2048 17, 16; 6000 39, 32; in
// four bits 14, 20; 18, 22; 28, 27; 65, 46.
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

template <bool F32, bool FOUR, int D, int STYLE>
void append_turned(const KvAppendLaunch& p, const Deal& d, hipStream_t stream)
{
    if (d.four_tokens)
        hipLaunchKernelGGL((kv_append_kernel<F32, FOUR, D, 4, STYLE>), d.grid, dim3(kThreads), 0, stream, p,
                           d.heads_part);
    else
        hipLaunchKernelGGL((kv_append_kernel<F32, FOUR, D, 1, STYLE>), d.grid, dim3(kThreads), 0, stream, p,
                           d.heads_part);
}

template <bool F32, bool FOUR, int D>
void append_to(const KvAppendLaunch& p, const Deal& d, hipStream_t stream)
{
    if (p.rope.axes == 0)
        append_turned<F32, FOUR, D, kStill>(p, d, stream);
    else if (p.rope.halves)
        append_turned<F32, FOUR, D, kHalves>(p, d, stream);
    else
        append_turned<F32, FOUR, D, kNeighbours>(p, d, stream);
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
