// C ABI of the key/value cache: the rotation's handle, and the checks of every
// descriptor before a kernel runs.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>
#include <string>

#include "awa_internal.h"
#include "kv_kernels.h"
#include "seedvr2_awa.h"

struct awa_rope
{
    awa::KvRope table;
    int rope_dim;
};

namespace
{

using awa::set_error;

int invalid(const std::string& message)
{
    set_error(message);
    return AWA_ERR_INVALID;
}

int launched(hipError_t e, const char* what)
{
    if (e == hipSuccess)
        return AWA_OK;
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return AWA_ERR_DEVICE;
}

bool aligned(const void* p, size_t bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Fills the kernels' view of the cache and of this call's `total` new rows.
int view(const awa_kv_cache* c, const awa_kv_rows* rows, int total, awa::KvView& out)
{
    if (!c || !rows)
        return invalid("null cache or rows");
    if (c->format != AWA_KV_BF16 && c->format != AWA_KV_MXFP4)
        return invalid("unknown cache format");
    if (c->head_dim != 64 && c->head_dim != 128)
        return invalid("the cache takes head_dim 64 or 128");
    if (c->page_tokens < 16 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
        return invalid("page_tokens must be a power of two from 16 to 1024");
    if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535)
        return invalid("the cache needs pages and 1 to 65535 heads");
    if (static_cast<long long>(c->pages) * c->kv_heads * c->page_tokens > 0x7fffffffll)
        return invalid("a pool has less than 2^31 rows");
    if (c->sequences <= 0 || c->sequences > 65535)
        return invalid("1 to 65535 sequences a call");
    if (c->table_width <= 0 || static_cast<long long>(c->table_width) * c->page_tokens > awa::kKvMaxSlots)
        return invalid("a page table row must name 1 to 2^30 slots");
    if (c->table_stride < c->table_width)
        return invalid("page table rows overlap");
    if (!c->k || !c->v || !c->page_table || !c->lengths)
        return invalid("null pool, page table or lengths");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->page_table, 4) || !aligned(c->lengths, 4) ||
        !aligned(c->status, 4) || !aligned(rows->cu_rows, 4))
        return invalid("pools must be 16-byte aligned, tables 4-byte aligned");
    if (c->format == AWA_KV_MXFP4 && (!c->k_scale || !c->v_scale || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)))
        return invalid("4-bit pages need 4-byte aligned scale pools");
    if (rows->max_rows <= 0 || rows->max_rows > awa::kKvMaxSlots)
        return invalid("max_rows must be 1 to 2^30");
    if (total > 1 << 25)
        return invalid("a call takes at most 2^25 rows");
    if (!rows->cu_rows && static_cast<long long>(rows->max_rows) * c->sequences != total)
        return invalid("without cu_rows the blobs must hold max_rows rows for every sequence");
    int shift = 0;
    while ((1 << shift) < c->page_tokens)
        shift++;
    out.pages = c->pages;
    out.page_shift = shift;
    out.heads = c->kv_heads;
    out.k = static_cast<unsigned char*>(c->k);
    out.v = static_cast<unsigned char*>(c->v);
    out.k_scale = static_cast<unsigned char*>(c->k_scale);
    out.v_scale = static_cast<unsigned char*>(c->v_scale);
    out.table = c->page_table;
    out.sequences = c->sequences;
    out.table_width = c->table_width;
    out.table_stride = c->table_stride;
    out.lengths = c->lengths;
    out.status = c->status;
    out.cu = rows->cu_rows;
    out.max_rows = rows->max_rows < total ? rows->max_rows : total;
    out.total_rows = total;
    return AWA_OK;
}

// A dims-3 Mat(head_dim, heads, rows) whose rows' starts are 16-byte aligned.
int row_blob(const awa_blob* b, const char* name, int head_dim, int heads, int rows, awa::KvRowsSource& out)
{
    if (!b || !b->data)
        return invalid(std::string(name) + ": null blob");
    if (b->dims != 3 || b->n != 1 || b->w != head_dim || b->h <= 0 || (heads > 0 && b->h != heads) || b->c <= 0 ||
        (rows > 0 && b->c != rows) || (b->elemsize != 2 && b->elemsize != 4) ||
        b->cstep < static_cast<long long>(b->w) * b->h)
        return invalid(std::string(name) + " must be an fp32 or bf16 Mat(head_dim, heads, rows)");
    if (!aligned(b->data, 16) || (b->cstep * b->elemsize) % 16)
        return invalid(std::string(name) + ": rows must start at 16-byte addresses");
    out.data = static_cast<const unsigned char*>(b->data);
    out.stride = b->cstep * b->elemsize;
    return AWA_OK;
}

int mask_rule(const awa_kv_mask* mask, awa::KvMaskRule& out)
{
    if (!mask)
        return invalid("null mask");
    if (mask->window < 0 || mask->sinks < 0 || mask->block < 1 || mask->max_length < 0 ||
        mask->window > awa::kKvMaxSlots || mask->sinks > awa::kKvMaxSlots || mask->block > awa::kKvMaxSlots)
        return invalid("mask: window and sinks are 0 to 2^30, block 1 to 2^30");
    out.window = mask->window;
    out.sinks = mask->sinks;
    out.block = mask->block;
    return AWA_OK;
}

// Everything of an attention call but the buffers it writes.
int attention(const awa_kv_cache* cache, const awa_kv_rows* rows, const awa_blob* q, const awa_kv_mask* mask,
              awa::KvAttentionLaunch& p)
{
    if (!cache)
        return invalid("null cache or rows");
    int rc = row_blob(q, "q", cache->head_dim, 0, 0, p.q);
    if (rc == AWA_OK)
        rc = view(cache, rows, q->c, p.cache);
    if (rc == AWA_OK)
        rc = mask_rule(mask, p.mask);
    if (rc != AWA_OK)
        return rc;
    if (q->h % cache->kv_heads)
        return invalid("query heads must be a multiple of the cache's heads");
    p.head_dim = cache->head_dim;
    const int group = q->h / cache->kv_heads;
    p.group = awa::kv_divisor(group);
    p.heads = awa::kv_divisor(q->h);
    p.f32 = q->elemsize == 4;
    p.four = cache->format == AWA_KV_MXFP4;
    const long long slots = static_cast<long long>(cache->table_width) * cache->page_tokens;
    const long long longest = mask->max_length > 0 && mask->max_length < slots ? mask->max_length : slots;
    if (static_cast<long long>(p.cache.max_rows) * q->h >= 1ll << 30)
        return invalid("max_rows times query heads must be below 2^30");
    awa::kv_attention_deal(p, static_cast<int>(longest));
    if (!awa::kv_attention_fits(p))
        return invalid("too many rows, heads and sequences for one call");
    return AWA_OK;
}

} // namespace

extern "C" {

int awa_rope_create(const awa_rope_desc* desc, awa_rope** rope)
{
    if (!desc || !rope)
        return invalid("null descriptor");
    *rope = nullptr;
    if (desc->axes < 1 || desc->axes > 4 || desc->rope_dim <= 0 || desc->rope_dim > 128 ||
        desc->rope_dim % (2 * desc->axes))
        return invalid("rope_dim must be 2 to 128 and a multiple of twice the 1 to 4 axes");
    if (desc->halves && (desc->axes != 1 || desc->rope_dim % 16))
        return invalid("halves need one axis and a rope_dim that is a multiple of 16");
    if (!desc->frequencies && !(std::isfinite(desc->base) && desc->base > 0.0))
        return invalid("the base must be positive");
    awa_rope* r = new (std::nothrow) awa_rope{};
    if (!r)
    {
        set_error("out of memory");
        return AWA_ERR_ALLOC;
    }
    r->rope_dim = desc->rope_dim;
    r->table.axes = desc->axes;
    r->table.pairs = desc->rope_dim / desc->axes / 2;
    r->table.halves = desc->halves ? 1 : 0;
    for (int i = 0; i < r->table.pairs; i++)
    {
        // Radians a position, then turns, whose whole part no angle needs.
        const long double f = desc->frequencies
                                  ? static_cast<long double>(desc->frequencies[i])
                                  : std::pow(static_cast<long double>(desc->base),
                                             -static_cast<long double>(i) / static_cast<long double>(r->table.pairs));
        long double turns = f / 6.283185307179586476925286766559L;
        turns -= std::floor(turns);
        if (!std::isfinite(turns))
        {
            delete r;
            return invalid("a frequency is not finite");
        }
        r->table.turns[i] = static_cast<unsigned long long>(std::ldexp(turns, 63)) << 1;
        r->table.turns[i] += std::ldexp(turns, 64) - static_cast<long double>(r->table.turns[i]) >= 1.0L ? 1 : 0;
    }
    *rope = r;
    return AWA_OK;
}

void awa_rope_destroy(awa_rope* rope)
{
    delete rope;
}

int awa_kv_append(const awa_kv_cache* cache, const awa_kv_rows* rows, const awa_blob* k, const awa_blob* v,
                  const awa_rope* rope, const int* positions, const awa_blob* q, const awa_blob* q_out, void* stream)
{
    awa::KvAppendLaunch p{};
    if (!cache)
        return invalid("null cache or rows");
    int rc = row_blob(k, "k", cache->head_dim, cache->kv_heads, 0, p.k);
    if (rc == AWA_OK)
        rc = row_blob(v, "v", cache->head_dim, cache->kv_heads, k->c, p.v);
    if (rc == AWA_OK)
        rc = view(cache, rows, k->c, p.cache);
    if (rc != AWA_OK)
        return rc;
    if (v->elemsize != k->elemsize)
        return invalid("k and v must be of one type");
    if ((q == nullptr) != (q_out == nullptr))
        return invalid("q and q_out come together");
    if (q)
    {
        if (!rope)
            return invalid("q is taken to be rotated: it needs a rope");
        rc = row_blob(q, "q", cache->head_dim, 0, k->c, p.q);
        if (rc == AWA_OK)
            rc = row_blob(q_out, "q_out", cache->head_dim, q->h, k->c, p.q_out);
        if (rc != AWA_OK)
            return rc;
        if (q->elemsize != k->elemsize || q_out->elemsize != k->elemsize)
            return invalid("q and q_out must be of k's type");
        p.q_heads = q->h;
        if (static_cast<long long>(q->h) + 2ll * cache->kv_heads >= 1 << 18)
            return invalid("too many heads");
    }
    if (rope)
    {
        if (rope->rope_dim > cache->head_dim)
            return invalid("rope_dim exceeds head_dim");
        if (!positions && rope->table.axes != 1)
            return invalid("a rope of several axes needs positions");
        if (!aligned(positions, 4))
            return invalid("positions must be 4-byte aligned");
        p.rope = rope->table;
    }
    p.positions = positions;
    p.head_dim = cache->head_dim;
    p.f32 = k->elemsize == 4;
    p.four = cache->format == AWA_KV_MXFP4;
    return launched(awa::launch_kv_append(p, static_cast<hipStream_t>(stream)), "kv append kernel launch");
}

int awa_kv_read(const awa_kv_cache* cache, const awa_kv_rows* rows, const awa_blob* k_out, const awa_blob* v_out,
                void* stream)
{
    awa::KvReadLaunch p{};
    if (!cache)
        return invalid("null cache or rows");
    int rc = row_blob(k_out, "k_out", cache->head_dim, cache->kv_heads, 0, p.k);
    if (rc == AWA_OK)
        rc = row_blob(v_out, "v_out", cache->head_dim, cache->kv_heads, k_out->c, p.v);
    if (rc == AWA_OK)
        rc = view(cache, rows, k_out->c, p.cache);
    if (rc != AWA_OK)
        return rc;
    if (v_out->elemsize != k_out->elemsize)
        return invalid("k_out and v_out must be of one type");
    p.head_dim = cache->head_dim;
    p.f32 = k_out->elemsize == 4;
    p.four = cache->format == AWA_KV_MXFP4;
    return launched(awa::launch_kv_read(p, static_cast<hipStream_t>(stream)), "kv read kernel launch");
}

int awa_kv_attention_workspace(const awa_kv_cache* cache, const awa_kv_rows* rows, const awa_blob* q,
                               const awa_kv_mask* mask, size_t* bytes)
{
    if (!bytes)
        return invalid("null bytes");
    awa::KvAttentionLaunch p{};
    const int rc = attention(cache, rows, q, mask, p);
    if (rc == AWA_OK)
        *bytes = awa::kv_attention_workspace_bytes(p);
    return rc;
}

int awa_kv_attention(const awa_kv_cache* cache, const awa_kv_rows* rows, const awa_blob* q, const awa_kv_mask* mask,
                     float scale, const awa_blob* out, void* workspace, size_t workspace_bytes, void* stream)
{
    awa::KvAttentionLaunch p{};
    int rc = attention(cache, rows, q, mask, p);
    if (rc == AWA_OK)
        rc = row_blob(out, "out", cache->head_dim, q->h, q->c, p.out);
    if (rc != AWA_OK)
        return rc;
    if (out->elemsize != q->elemsize)
        return invalid("out must be of q's type");
    if (!std::isfinite(scale))
        return invalid("the scale must be finite");
    p.scale_log2 = scale * 1.44269504088896340736f;
    const size_t need = awa::kv_attention_workspace_bytes(p);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return invalid("this call needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    awa::kv_attention_set_workspace(p, workspace);
    return launched(awa::launch_kv_attention(p, static_cast<hipStream_t>(stream)), "kv attention kernel launch");
}

// What a row sees and how rows and keys are dealt out, on the host (tests).
int awa_kv_host_sequence(int first, int end, int length, int capacity, int max_rows, int total_rows, int* out)
{
    const awa::KvSequence s = awa::kv_sequence(first, end, length, capacity, max_rows, total_rows);
    out[0] = s.first, out[1] = s.rows, out[2] = s.length, out[3] = static_cast<int>(s.bad);
    return AWA_OK;
}

int awa_kv_host_divide(int n, int d)
{
    return awa::kv_divide(n, awa::kv_divisor(d));
}

int awa_kv_host_span(int window, int sinks, int block, int slot, int length, int* out)
{
    const awa::KvSpan s = awa::kv_span({window, sinks, block}, slot, length);
    out[0] = s.sinks, out[1] = s.begin, out[2] = s.end;
    return AWA_OK;
}

int awa_kv_host_tiles(const int* first, const int* last, int shift, int* out)
{
    const awa::KvTiles t = awa::kv_tiles({first[0], first[1], first[2]}, {last[0], last[1], last[2]}, shift);
    out[0] = t.sinks, out[1] = t.begin, out[2] = t.rest;
    return AWA_OK;
}

} // extern "C"
