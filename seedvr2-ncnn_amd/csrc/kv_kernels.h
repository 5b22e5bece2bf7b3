// Key/value cache in pages: the launch interface of its kernels (gfx950) and
// the arithmetic that kernels and host checks share: which rows a sequence
// brings, what a row sees, and how its keys are dealt out. Pointers are device
// pointers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "seedvr2_awa.h"

namespace awa
{

constexpr int kKvMaxSlots = 1 << 30; // slots a page table row may name
constexpr int kKvGroup = 32;         // features that share a 4-bit row's power of two
constexpr int kRopeMaxPairs = 64;

struct KvView
{
    int pages, page_shift, heads; // key/value heads
    unsigned char *k, *v, *k_scale, *v_scale;
    const int* table;
    int sequences, table_width, table_stride;
    const int* lengths;
    int* status;
    // This call's new rows.
    const int* cu;
    int max_rows, total_rows;
};

// floor(n / d) for 0 <= n < 2^30 as a multiplication: with 2^(s - 1) < d <= 2^s
// and m = floor(2^(30 + s) / d) + 1, m d is above 2^(30 + s) by at most 2^s, so
// that n m / 2^(30 + s) is above n / d by less than 1 / d.
struct KvDivisor
{
    unsigned m;
    int shift, d;
};

__host__ inline KvDivisor kv_divisor(int d)
{
    int s = 0;
    while ((1ll << s) < d)
        s++;
    return {static_cast<unsigned>((1ull << (30 + s)) / d + 1), 30 + s, d};
}

__host__ __device__ inline int kv_divide(int n, const KvDivisor& by)
{
    return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(n)) * by.m) >> by.shift);
}

// The new rows of one sequence: packed rows [first, first + rows), at slots
// [length - rows, length). What does not fit together (bad != 0) has no rows,
// so that nothing of it is read or written.
struct KvSequence
{
    int first, rows, length;
    unsigned bad;
};

__host__ __device__ inline KvSequence kv_sequence(int first, int end, int length, int capacity, int max_rows,
                                                  int total_rows)
{
    KvSequence s{first, 0, length, 0u};
    if (first < 0 || end < first || end > total_rows || end - first > max_rows)
        s.bad |= AWA_KV_BAD_ROWS;
    if (length < 0 || length > capacity || (!s.bad && end - first > length))
        s.bad |= AWA_KV_BAD_LENGTH;
    if (!s.bad)
        s.rows = end - first;
    return s;
}

__host__ __device__ inline KvSequence kv_sequence(const KvView& c, int s)
{
    const int first = c.cu ? c.cu[s] : s * c.max_rows;
    const int end = c.cu ? c.cu[s + 1] : first + c.max_rows;
    return kv_sequence(first, end, c.lengths[s], c.table_width << c.page_shift, c.max_rows, c.total_rows);
}

struct KvMaskRule
{
    int window, sinks, block;
};

// What the row at slot p of a sequence of `length` sees: keys [0, sinks) and
// [begin, end), sinks <= begin <= end. All three grow with p.
struct KvSpan
{
    int sinks, begin, end;
};

__host__ __device__ inline KvSpan kv_span(const KvMaskRule& m, int p, int length)
{
    long long e = static_cast<long long>(p) + 1;
    if (m.block > 1)
    {
        // The end of the row's block; blocks are counted from slot `sinks`.
        const int d = p + 1 - m.sinks;
        const int q = d >= 0 ? (d + m.block - 1 < 0 ? d / m.block + (d % m.block != 0) : (d + m.block - 1) / m.block)
                             : -(-d / m.block);
        e = m.sinks + static_cast<long long>(q) * m.block;
    }
    KvSpan s;
    s.end = static_cast<int>(e < length ? e : length);
    const long long b = m.window > 0 && e > m.window ? e - m.window : 0;
    s.begin = static_cast<int>(b < s.end ? b : s.end);
    s.sinks = m.sinks < s.begin ? m.sinks : s.begin;
    return s;
}

// The key tiles that rows from `first` to `last` (spans of the first and the
// last row) see: tiles [0, sinks) and [begin, begin + rest).
struct KvTiles
{
    int sinks, begin, rest;
};

__host__ __device__ inline KvTiles kv_tiles(const KvSpan& first, const KvSpan& last, int tile_shift)
{
    const int up = (1 << tile_shift) - 1;
    KvTiles t;
    t.sinks = (last.sinks + up) >> tile_shift;
    t.begin = first.begin >> tile_shift;
    if (t.begin < t.sinks)
        t.begin = t.sinks;
    const int end = (last.end + up) >> tile_shift;
    t.rest = end > t.begin ? end - t.begin : 0;
    return t;
}

// Rotation of the first rope_dim features of a row.
struct KvRope
{
    // Turns a position, as a 64-bit fraction: the angle of position x is
    // 2 pi (x * turns mod 2^64) / 2^64, exact for every 32-bit x.
    unsigned long long turns[kRopeMaxPairs];
    int pairs;      // pairs an axis
    int axes;       // 0: no rotation
    int halves;     // pair i is features i and i + pairs, else 2 i and 2 i + 1
};

struct KvRowsSource
{
    const unsigned char* data;
    long long stride; // bytes from row to row
};

struct KvAppendLaunch
{
    KvView cache;
    int head_dim, q_heads;
    bool f32;  // type of q, k, v and q_out
    bool four; // 4-bit pages
    KvRowsSource q, k, v, q_out; // q.data null: none
    const int* positions;        // null: the slot
    KvRope rope;
};
hipError_t launch_kv_append(const KvAppendLaunch& p, hipStream_t stream);

struct KvReadLaunch
{
    KvView cache;
    int head_dim;
    bool f32; // type of k and v
    bool four;
    KvRowsSource k, v;
};
hipError_t launch_kv_read(const KvReadLaunch& p, hipStream_t stream);

// How the key tiles of a row tile are dealt out: parts of part_tiles (the last
// takes what lengths have beyond their bound).
struct KvParts
{
    int splits, part_tiles;
    int tiles; // the first row tiles of a sequence that are split; later ones are not
    // splits > 1: of every part the rows [D], unnormalised and relative to their
    // maximum, by row and query head, then all (maximum, sum) pairs.
    float* partial;
    int seq_rows;   // rows that a sequence has room for, 0: as packed
    long long rows; // of all sequences
};

struct KvAttentionLaunch
{
    KvView cache;
    int head_dim;
    KvDivisor group; // query heads a key/value head
    KvDivisor heads; // query heads
    bool f32, four;
    KvRowsSource q, out;
    KvMaskRule mask;
    float scale_log2; // softmax scale * log2 e
    bool few;         // rows: row tiles of 16, else of 128
    bool wide;        // few: eight waves a workgroup, not four
    int tiles;        // row tiles of the longest sequence
    // Of sequences of one tile of 128 rows, and of longer ones.
    KvParts one, more;
    // Where many sequences are far shorter than the longest, the parts of all of
    // them are numbered through, `parts` at most: first those of longer
    // sequences, then those of one tile. Of both the number of the first part by
    // sequence, [2][sequences + 1].
    bool listed;
    long long parts; // else: of every sequence
    int* list;
};

// Fills in how the work is dealt out (few and below). max_length: a bound of
// the lengths.
void kv_attention_deal(KvAttentionLaunch& p, int max_length);
bool kv_attention_fits(const KvAttentionLaunch& p); // its grids can be launched
// Bytes of the list and of `one` and `more`'s parts, and where they are.
size_t kv_attention_workspace_bytes(const KvAttentionLaunch& p);
void kv_attention_set_workspace(KvAttentionLaunch& p, void* workspace);
hipError_t launch_kv_attention(const KvAttentionLaunch& p, hipStream_t stream);

} // namespace awa
