// extern "C" entry points between a layer's projections: rotary positions, the paged cache, attention.  Argument checks and
// the choice of kernels; nothing here allocates, synchronises or throws.
#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdint.h>

#include "attention.hpp"
#include "attention_shared.hpp"
#include "head_rotary.hpp"

namespace sngguf {
int launch_attention_rows(const AttentionArgs& a, int rows, int dim, bool q8, hipStream_t stream);
int launch_attention_tiles(const AttentionArgs& a, int rows, int dim, int source, hipStream_t stream);
}  // namespace sngguf

namespace {

using sngguf::AttentionArgs;
using sngguf::bf16_t;
using sngguf::RotaryCacheArgs;

constexpr int64_t kMost = (int64_t)1 << 31;           // tokens, heads, pages: numbered with 32 bits
constexpr int64_t kMostStride = (int64_t)1 << 26;     // elements between tokens: sixteen rows within 32-bit byte offsets

// Threads of a launch are numbered with 32 bits.
bool launch_fits(int64_t workgroups, int64_t threads) { return workgroups < kMost && workgroups * threads < (int64_t)1 << 32; }

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_cache(const sngguf_kv_cache* c) {
    if (!c) return SNGGUF_E_NULLPTR;
    if (c->qtype != SNGGUF_TYPE_BF16 && c->qtype != SNGGUF_TYPE_Q8_0) return SNGGUF_E_BADTYPE;
    if (c->pages < 1 || c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)) != 0 || c->pages >= kMost ||
        c->kv_heads < 1 || c->kv_heads > 65535 || c->dim < 32 || c->dim > 256 || c->dim % 32 != 0)
        return SNGGUF_E_BADSHAPE;
    if (!c->k || !c->v) return SNGGUF_E_NULLPTR;
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return SNGGUF_E_ALIGN;
    if (c->qtype == SNGGUF_TYPE_Q8_0) {
        if (!c->k_scale || !c->v_scale) return SNGGUF_E_NULLPTR;
        if (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16)) return SNGGUF_E_ALIGN;
    }
    return SNGGUF_OK;
}

int log2_of(int64_t v) {
    int s = 0;
    while (((int64_t)1 << s) < v) s++;
    return s;
}

void set_cache(RotaryCacheArgs& a, const sngguf_kv_cache* c) {
    a.k_pages = c->k;
    a.v_pages = c->v;
    a.k_scales = static_cast<uint16_t*>(c->k_scale);
    a.v_scales = static_cast<uint16_t*>(c->v_scale);
    a.page_shift = log2_of(c->page_size);
    a.slot_count = c->pages * c->page_size;
    a.kv_heads = (int32_t)c->kv_heads;
}

// Rows of whole 16-byte pieces
bool whole_pieces(const void* p, int64_t token, int64_t head) { return aligned(p, 16) && token % 8 == 0 && head % 8 == 0; }

int check_table(const sngguf_rotary_table* t, const int64_t* positions, int64_t tokens, int64_t dim, int64_t heads) {
    if (!t) return SNGGUF_E_NULLPTR;
    if (tokens < 0 || tokens >= kMost || dim < 8 || dim > 1024 || dim % 8 != 0 || heads < 1 || heads > 65535 || t->pairs < 1 || 2 * t->pairs > dim ||
        !isfinite(t->magnitude))
        return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!t->turns || !positions) return SNGGUF_E_NULLPTR;
    if (!aligned(t->turns, 8) || !aligned(positions, 8)) return SNGGUF_E_ALIGN;
    return SNGGUF_OK;
}

void set_table(RotaryCacheArgs& a, const sngguf_rotary_table* t, const int64_t* positions) {
    a.turns = t->turns;
    a.magnitude = t->magnitude;
    a.positions = positions;
    a.pairs = (int32_t)t->pairs;
    a.interleaved = t->interleaved != 0;
}

int check_axes(const sngguf_rotary_axes* t, const int64_t* positions, int64_t axes, int64_t tokens, int64_t dim, int64_t heads) {
    if (!t) return SNGGUF_E_NULLPTR;
    if (tokens < 0 || tokens >= kMost || dim < 8 || dim > 512 || dim % 8 != 0 || heads < 1 || heads > 65535 || t->pairs < 1 || 2 * t->pairs > dim ||
        !isfinite(t->magnitude) || t->parts < 1 || t->parts > sngguf::kMostParts || axes < 1 || axes >= kMost)
        return SNGGUF_E_BADSHAPE;
    int64_t elements = 0;
    for (int p = 0; p < t->parts; p++) {
        if (t->part[p] < 2 || t->part[p] > dim || t->part[p] % 2 != 0) return SNGGUF_E_BADSHAPE;
        elements += t->part[p];
    }
    if (elements != 2 * t->pairs) return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!t->turns || !positions) return SNGGUF_E_NULLPTR;
    if (!aligned(t->turns, 8) || !aligned(positions, 8) || !aligned(t->axis, 4)) return SNGGUF_E_ALIGN;
    return SNGGUF_OK;
}

int check_norm(const sngguf_head_norm* n, int64_t dim) {
    if (!n) return SNGGUF_OK;
    if (n->weight_type != 0 && n->weight_type != 2) return SNGGUF_E_BADTYPE;
    if (n->parts < 1 || n->parts > sngguf::kMostParts || !(n->eps >= 0.f) || !isfinite(n->eps)) return SNGGUF_E_BADSHAPE;
    int64_t elements = 0;
    for (int p = 0; p < n->parts; p++) {
        if (n->elements[p] < 8 || n->elements[p] > dim || n->elements[p] % 8 != 0) return SNGGUF_E_BADSHAPE;
        elements += n->elements[p];
    }
    if (elements != dim) return SNGGUF_E_BADSHAPE;
    for (int p = 0; p < n->parts; p++) {
        if (!n->weight[p]) return SNGGUF_E_NULLPTR;
        if (!aligned(n->weight[p], 16)) return SNGGUF_E_ALIGN;
    }
    return SNGGUF_OK;
}

void set_norm(sngguf::HeadNormArgs& a, const sngguf_head_norm* n) {
    if (!n) return;
    a.parts = n->parts;
    a.bf16 = n->weight_type == 2;
    a.eps = n->eps;
    for (int p = 0; p < n->parts; p++) {
        a.weight[p] = n->weight[p];
        a.elements[p] = n->elements[p];
        a.one_over[p] = 1.f / (float)n->elements[p];
    }
}

void set_axes(sngguf::HeadRotaryArgs& a, const sngguf_rotary_axes* t, const int64_t* positions, int64_t axes, int64_t axis_stride) {
    a.turns = t->turns;
    a.axis = t->axis;
    a.magnitude = t->magnitude;
    a.positions = positions;
    a.axes = (int32_t)axes;
    a.axis_stride = axis_stride;
    a.pairs = (int32_t)t->pairs;
    a.interleaved = t->interleaved != 0;
    a.parts = t->parts;
    for (int p = 0; p < t->parts; p++) a.part[p] = t->part[p];
}

// ---- attention: how much is launched ----------------------------------------------------------------------------------

constexpr int64_t kMostKeys = kMost - 65536;          // of a sequence: a few tiles more still have 32-bit numbers

constexpr int kRowsLeast = 2, kRowsKeys = 128;        // key tiles that a split has at least; keys of a tile
constexpr int kTilesLeast = 16, kTilesKeys = 64;     // (a workgroup costs as much as five tiles before its first and behind its last)
// The same for keys that sequences have in common, whose rows have no other work (64 over 4096 / 16 over 16384 / 200 over 2048 tokens, bf16, with
// 2: 52.4 / 42.4 / 59.5 us, 4: 49.6 / 42.7 / 59.1, 8: 53.5 / 41.6 / 60.7, 16: 61.8 / 50.2 / 70.3)
constexpr int kCommonLeast = 4;

int kernel_dim(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// The kernel for many rows, bound by its arithmetic, has two more
int many_dim(int64_t dim) { return dim > 64 && dim <= 96 ? 96 : dim > 128 && dim <= 192 ? 192 : kernel_dim(dim); }

// Workgroups that the device's 256 compute units take at a time, by the registers of the kernels
int few_at_a_time(int rows, int dim) { return rows * dim <= 16 * 128 ? 768 : rows * dim <= 16 * 256 && dim < 256 ? 512 : 256; }
int many_at_a_time(int rows, int dim) { return rows == 128 && dim <= 128 ? 512 : 256; }

struct Launch {
    int rows;              // of a tile
    int64_t tiles;         // (row tile, head) pairs at most
    int32_t want;          // workgroups aimed at where keys are split
    int64_t grid, partial_bytes;
};

// Split only where unsplit workgroups leave compute units idle, and `least` tiles of keys can be had for two.
Launch plan(int64_t tiles, int64_t keys, int dim, int rows, int want, int64_t least) {
    Launch p;
    p.rows = rows;
    p.tiles = tiles;
    p.want = want;
    const bool split = tiles < want && keys >= 2 * least;
    p.grid = tiles + (split ? want : 0);
    p.partial_bytes = split ? p.grid * rows * (dim + 2) * 4 : 0;
    return p;
}

// Row tiles of all sequences at most: every sequence's last one may hold a single row
int64_t row_tiles(int64_t tokens, int64_t sequences, int64_t group, int rows) { return (tokens * group + sequences * (rows - 1)) / rows; }

// The kernel for many rows: 256 a workgroup (eight wavefronts that share tiles), or 128 where a sequence's only tile would be
// mostly empty, or where 256-row workgroups leave two of five compute units idle and there are no keys to split (one prompt
// of 1024 tokens and 8 heads of keys: 29 us against 33; of 1500: 43 against 42; of 4096: 150 against 135).
// Workgroups of equal work that leave a last round nearly empty are not split: 2500 queries over 3000 keys, 320 workgroups, took 193 us
// as 960 instead of 173.
Launch plan_many(int64_t tokens, int64_t keys, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim) {
    const int d = kernel_dim(dim);
    const int64_t group = heads / kv_heads, key_tiles = keys / kTilesKeys + 1;
    const bool wide = many_dim(dim) <= 192 && tokens * group >= 512 * sequences &&
                      (key_tiles >= 2 * kTilesLeast || kv_heads * row_tiles(tokens, sequences, group, 256) >= 160);
    const int rows = wide ? 256 : 128;
    return plan(kv_heads * row_tiles(tokens, sequences, group, rows), key_tiles, d, rows, many_at_a_time(rows, d), kTilesLeast);
}

struct PagedPlan {
    bool few, many;        // which kernels run
    int64_t few_rows;      // sequences of at most so many rows go to the first
    int64_t most_rows;     // of a tile of the first, as far as is known
    Launch a, b;
};

PagedPlan paged_plan(int64_t tokens, int64_t sequences, int64_t max_new, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    PagedPlan p;
    const int64_t group = heads / kv_heads;
    const int64_t most = (max_new > 0 && max_new < tokens ? max_new : tokens) * group;
    // a tile of 64 rows leaves a SIMD one wavefront: it pays where sequences are few and their keys split finer than the other kernel's
    // (16 new tokens of 4 heads a group, caches in turn, 8 bits / bf16: one sequence of 30000 45 / 44 us against 73 / 74, four of 8000
    // 53 / 52 against 56 / 55, eight 82 / 83 against 72 / 73, sixteen 142 / 149 against 118 / 121)
    const int d = kernel_dim(dim), widest = d == 256 || sequences * kv_heads > 32 ? 32 : 64;
    // one kernel where no sequence has more rows than its tile; else single tokens and chunks each have their own
    const int64_t r = most <= widest ? most : group;
    const int rows = r <= 16 ? 16 : r <= 32 ? 32 : widest;
    p.few = r <= widest;
    p.many = most > widest;
    p.few_rows = !p.many ? kMost - 1 : p.few ? rows : 0;
    p.most_rows = most < rows ? most : rows;
    const int64_t tiles = kv_heads * (p.many ? sequences : row_tiles(tokens, sequences, group, rows));
    p.a = plan(tiles, keys / kRowsKeys + 1, d, rows, few_at_a_time(rows, d), kRowsLeast);
    p.b = plan_many(tokens, keys, sequences, heads, kv_heads, dim);
    return p;
}

bool heads_fit(int64_t heads, int64_t kv_heads, int64_t dim) {
    return heads >= 1 && heads <= 65535 && kv_heads >= 1 && heads % kv_heads == 0 && dim >= 32 && dim <= 256 && dim % 32 == 0;
}

int launch_many(AttentionArgs& a, const Launch& p, int dim, int source, float* partial, hipStream_t stream) {
    const int64_t most_rows = a.tokens_q * a.group;
    a.partial = partial;
    a.want = p.want;
    a.least = kTilesLeast;
    a.grid = partial ? p.grid : p.tiles;
    const int rc = sngguf::launch_attention_tiles(a, p.rows, many_dim(a.dim), source, stream);
    if (rc != SNGGUF_OK || !partial) return rc;
    return sngguf::launch_attention_combine(a, p.rows, kTilesKeys, dim, p.tiles, most_rows, stream);
}

// ---- sequences that begin alike ----------------------------------------------------------------------------------------

// The launches of partial results (common keys that many rows see; few rows; many rows), and where everything lies in the workspace
struct SharedPlan {
    Launch launch[sngguf::kSharedLaunches];
    int32_t few_rows;      // sequences of at most so many rows go to that kernel
    int64_t entries, sequence_of, map[sngguf::kSharedLaunches], partial[sngguf::kSharedLaunches], bytes;
};

// Whether what sequences have in common is left to each of them, as by sngguf_paged_attention:
//  * where they can have few keys together, the plan and the join cost more than reading the common ones again from the caches (32 / 8 heads of
//    128, bf16, 8 sequences of 4300 keys at most 23.5 us against 22.2, 32 of 1250 22.8 against 25.9, 64 of 700 25.0 against 26.7; 8 bits, 8 of 4300
//    23.4 against 21.5, 4 of 16600 30.1 against 30.8);
//  * where they have 256 rows each on average, whose tiles are full already (two of 256 tokens and four of one, 6016 keys in common: 107 us against 96).
//    An average: a prompt of some thousand tokens among single tokens sends these there as well, which then read what is common each by itself.
bool shared_alone(int64_t tokens, int64_t sequences, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    return (double)sequences * (double)keys * (double)(kv_heads * dim) < (double)(40 << 20) || tokens * (heads / kv_heads) >= 256 * sequences;
}

SharedPlan shared_plan(int64_t tokens, int64_t sequences, int64_t groups, int64_t max_new, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, bool q8) {
    SharedPlan p = {};
    const int64_t group = heads / kv_heads;
    const int d = kernel_dim(dim);
    // Room for every row tile and, where keys are split, for `want` workgroups more.  With c key tiles a split, an entry of r row tiles and k key tiles takes
    // r ceil(k / c) <= r k / c + r (1 - 1 / c) workgroups, and c is chosen for a sum of r k / c of no more than `want`, within
    // 1e-5 of it: over all entries, being whole, no more than want + row tiles.  An entry that found no room would be passed over by the join.
    auto planned = [&](int64_t tiles, int rows, int want, int64_t key_tiles, int64_t least) {
        Launch x;
        x.rows = rows;
        x.tiles = tiles;
        x.want = key_tiles >= 2 * least ? want : 0;
        x.grid = (tiles + (x.want + kv_heads - 1) / kv_heads) * kv_heads;     // (tiles here: of a key / value head)
        x.partial_bytes = x.grid * rows * (d + 2) * 4;
        return x;
    };
    // All queries of a group are rows of its common keys.  While rows x keys are few, these go to the kernel for few rows, in one launch and in the
    // same tiles as what sequences have of their own: tiles read the common keys again, from the caches, but there is a launch less, and more
    // wavefronts than with larger tiles.  bf16, 16 sequences of 4 heads a group over 8192 / 16384 / 32768 common keys 31.7 / 44.6 / 75.9 us
    // against 36.4 / 43.3 / 56.2, 64 over 512 / 2048 25.0 / 40.8 against 37.9 / 41.4; 8 bits, 16 over 16384 / 32768 39.2 / 54.6 against 45.1 /
    // 54.6, 32 over 8192 / 16384 40.1 / 55.3 against 43.9 / 51.4.
    // (As tiles of 32 rows, the common keys read half as often: 8 bits 3 us less to 1 more, bf16 level to 6 more; of 64 rows 7 to 30 more.)
    const PagedPlan own = paged_plan(tokens, sequences, max_new, keys, heads, kv_heads, dim);
    const int64_t mean = tokens * group / groups;
    const bool few_common = own.few && (double)mean * (double)keys <= (q8 ? 1.5 : 0.875) * (double)(1 << 20);
    p.few_rows = (int32_t)own.few_rows;
    const int rows = own.a.rows;
    if (own.few)
        p.launch[1] = planned((own.many ? sequences : row_tiles(tokens, sequences, group, rows)) + (few_common ? row_tiles(tokens, groups, group, rows) : 0), rows, own.a.want,
                              keys / kRowsKeys + 1, kRowsLeast);
    if (own.many) p.launch[2] = planned(row_tiles(tokens, sequences, group, own.b.rows), own.b.rows, own.b.want, keys / kTilesKeys + 1, kTilesLeast);
    // Else 128 or 256 rows a workgroup: 64 / 128 sequences over 16384 / 8192 in bf16 60.6 / 72.6 us with 256, 63.9 / 74.5 with 128; 64 over 4096 49.5
    // against 46.7; 8 bits level.
    if (!few_common) {
        const int many = many_dim(dim) <= 192 && mean > 128 ? 256 : 128;
        p.launch[0] = planned(row_tiles(tokens, groups, group, many), many, many_at_a_time(many, d), keys / kTilesKeys, kCommonLeast);
    }
    auto room = [&](int64_t bytes) {
        const int64_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    p.entries = room((groups + sequences) * (int64_t)sizeof(sngguf::AttentionEntry));
    p.sequence_of = room(tokens * 4);
    for (int l = 0; l < sngguf::kSharedLaunches; l++) p.map[l] = room(p.launch[l].grid / kv_heads * (int64_t)sizeof(sngguf::AttentionEntry));
    for (int l = 0; l < sngguf::kSharedLaunches; l++) p.partial[l] = room(p.launch[l].partial_bytes);
    return p;
}

bool shared_sizes_fit(int64_t tokens, int64_t sequences, int64_t groups, int64_t max_new, int64_t keys) {
    return tokens > 0 && tokens < kMost && sequences > 0 && groups > 0 && sequences + groups < kMost / 64 && max_new >= 0 && keys >= 0 && keys <= kMostKeys;
}

}  // namespace

extern "C" {

int sngguf_rotary(const sngguf_rotary_table* table, const int64_t* positions, int64_t tokens, int64_t dim, const void* q,
                  int64_t q_heads, int64_t q_token, int64_t q_head, void* q_out, int64_t q_out_token, int64_t q_out_head,
                  const void* k, int64_t k_heads, int64_t k_token, int64_t k_head, void* k_out, int64_t k_out_token,
                  int64_t k_out_head, void* stream) {
    const int rc = check_table(table, positions, tokens, dim, q_heads);
    if (rc != SNGGUF_OK) return rc;
    if (k_heads < 0 || k_heads > 65535) return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!q || !q_out || (k_heads && (!k || !k_out))) return SNGGUF_E_NULLPTR;
    if (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(k, 2) || !aligned(k_out, 2)) return SNGGUF_E_ALIGN;
    RotaryCacheArgs a = {};
    set_table(a, table, positions);
    a.q = static_cast<const bf16_t*>(q);
    a.q_out = static_cast<bf16_t*>(q_out);
    a.k = static_cast<const bf16_t*>(k);
    a.k_out = static_cast<bf16_t*>(k_out);
    a.q_token = q_token, a.q_head = q_head, a.q_out_token = q_out_token, a.q_out_head = q_out_head;
    a.k_token = k_token, a.k_head = k_head, a.k_out_token = k_out_token, a.k_out_head = k_out_head;
    a.tokens = tokens;
    a.dim = (int32_t)dim;
    a.q_heads = (int32_t)q_heads;
    a.k_heads = (int32_t)k_heads;
    a.wide = whole_pieces(q, q_token, q_head) && whole_pieces(q_out, q_out_token, q_out_head) &&
             (!k_heads || (whole_pieces(k, k_token, k_head) && whole_pieces(k_out, k_out_token, k_out_head)));
    return sngguf::launch_rotary_cache(a, 0, static_cast<hipStream_t>(stream));
}

int sngguf_cache_write(const sngguf_kv_cache* cache, const void* k, int64_t k_token, int64_t k_head, const void* v,
                       int64_t v_token, int64_t v_head, const int64_t* slots, int64_t tokens, void* stream) {
    const int rc = check_cache(cache);
    if (rc != SNGGUF_OK) return rc;
    if (tokens < 0 || tokens >= kMost) return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!k || !v || !slots) return SNGGUF_E_NULLPTR;
    if (!aligned(k, 2) || !aligned(v, 2) || !aligned(slots, 8)) return SNGGUF_E_ALIGN;
    RotaryCacheArgs a = {};
    set_cache(a, cache);
    a.k = static_cast<const bf16_t*>(k);
    a.v = static_cast<const bf16_t*>(v);
    a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
    a.slots = slots;
    a.tokens = tokens;
    a.dim = (int32_t)cache->dim;
    a.wide = whole_pieces(k, k_token, k_head) && whole_pieces(v, v_token, v_head);
    return sngguf::launch_rotary_cache(a, cache->qtype == SNGGUF_TYPE_Q8_0 ? 2 : 1, static_cast<hipStream_t>(stream));
}

int sngguf_cache_write_rotary(const sngguf_kv_cache* cache, const sngguf_rotary_table* table, const int64_t* positions,
                              const void* q, int64_t q_heads, int64_t q_token, int64_t q_head, void* q_out, int64_t q_out_token,
                              int64_t q_out_head, const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                              int64_t v_head, const int64_t* slots, int64_t tokens, void* stream) {
    int rc = check_cache(cache);
    if (rc == SNGGUF_OK) rc = check_table(table, positions, tokens, cache->dim, q_heads);
    if (rc != SNGGUF_OK || tokens == 0) return rc;
    if (!q || !q_out || !k || !v || !slots) return SNGGUF_E_NULLPTR;
    if (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(slots, 8)) return SNGGUF_E_ALIGN;
    RotaryCacheArgs a = {};
    set_cache(a, cache);
    set_table(a, table, positions);
    a.q = static_cast<const bf16_t*>(q);
    a.q_out = static_cast<bf16_t*>(q_out);
    a.k = static_cast<const bf16_t*>(k);
    a.v = static_cast<const bf16_t*>(v);
    a.q_token = q_token, a.q_head = q_head, a.q_out_token = q_out_token, a.q_out_head = q_out_head;
    a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
    a.slots = slots;
    a.tokens = tokens;
    a.dim = (int32_t)cache->dim;
    a.q_heads = (int32_t)q_heads;
    a.wide = whole_pieces(q, q_token, q_head) && whole_pieces(q_out, q_out_token, q_out_head) && whole_pieces(k, k_token, k_head) &&
             whole_pieces(v, v_token, v_head);
    return sngguf::launch_rotary_cache(a, cache->qtype == SNGGUF_TYPE_Q8_0 ? 2 : 1, static_cast<hipStream_t>(stream));
}

int sngguf_head_rotary(const sngguf_rotary_axes* table, const int64_t* positions, int64_t axes, int64_t axis_stride, int64_t tokens, int64_t dim,
                       const sngguf_head_norm* q_norm, const void* q, int64_t q_heads, int64_t q_token, int64_t q_head, void* q_out,
                       int64_t q_out_token, int64_t q_out_head, const sngguf_head_norm* k_norm, const void* k, int64_t k_heads, int64_t k_token,
                       int64_t k_head, void* k_out, int64_t k_out_token, int64_t k_out_head, void* stream) {
    int rc = check_axes(table, positions, axes, tokens, dim, q_heads);
    if (rc == SNGGUF_OK) rc = check_norm(q_norm, dim);
    if (rc == SNGGUF_OK) rc = check_norm(k_norm, dim);
    if (rc != SNGGUF_OK) return rc;
    if (k_heads < 0 || k_heads > 65535) return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!q || !q_out || (k_heads && (!k || !k_out))) return SNGGUF_E_NULLPTR;
    if (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(k, 2) || !aligned(k_out, 2)) return SNGGUF_E_ALIGN;
    sngguf::HeadRotaryArgs a = {};
    set_axes(a, table, positions, axes, axis_stride);
    set_norm(a.q_norm, q_norm);
    if (k_heads) set_norm(a.k_norm, k_norm);
    a.q = static_cast<const bf16_t*>(q);
    a.q_out = static_cast<bf16_t*>(q_out);
    a.k = static_cast<const bf16_t*>(k);
    a.k_out = static_cast<bf16_t*>(k_out);
    a.q_token = q_token, a.q_head = q_head, a.q_out_token = q_out_token, a.q_out_head = q_out_head;
    a.k_token = k_token, a.k_head = k_head, a.k_out_token = k_out_token, a.k_out_head = k_out_head;
    a.tokens = tokens;
    a.dim = (int32_t)dim;
    a.q_heads = (int32_t)q_heads;
    a.k_heads = (int32_t)k_heads;
    a.wide = whole_pieces(q, q_token, q_head) && whole_pieces(q_out, q_out_token, q_out_head) &&
             (!k_heads || (whole_pieces(k, k_token, k_head) && whole_pieces(k_out, k_out_token, k_out_head)));
    return sngguf::launch_head_rotary(a, 0, static_cast<hipStream_t>(stream));
}

int sngguf_cache_write_head_rotary(const sngguf_kv_cache* cache, const sngguf_rotary_axes* table, const int64_t* positions, int64_t axes,
                                   int64_t axis_stride, const sngguf_head_norm* q_norm, const void* q, int64_t q_heads, int64_t q_token,
                                   int64_t q_head, void* q_out, int64_t q_out_token, int64_t q_out_head, const sngguf_head_norm* k_norm,
                                   const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                                   const int64_t* slots, int64_t tokens, void* stream) {
    int rc = check_cache(cache);
    if (rc == SNGGUF_OK) rc = check_axes(table, positions, axes, tokens, cache->dim, q_heads);
    if (rc == SNGGUF_OK) rc = check_norm(q_norm, cache->dim);
    if (rc == SNGGUF_OK) rc = check_norm(k_norm, cache->dim);
    if (rc != SNGGUF_OK || tokens == 0) return rc;
    if (!q || !q_out || !k || !v || !slots) return SNGGUF_E_NULLPTR;
    if (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(slots, 8)) return SNGGUF_E_ALIGN;
    sngguf::HeadRotaryArgs a = {};
    set_cache(a, cache);
    set_axes(a, table, positions, axes, axis_stride);
    set_norm(a.q_norm, q_norm);
    set_norm(a.k_norm, k_norm);
    if (cache->qtype != SNGGUF_TYPE_Q8_0) a.k_scales = a.v_scales = nullptr;
    a.q = static_cast<const bf16_t*>(q);
    a.q_out = static_cast<bf16_t*>(q_out);
    a.k = static_cast<const bf16_t*>(k);
    a.v = static_cast<const bf16_t*>(v);
    a.q_token = q_token, a.q_head = q_head, a.q_out_token = q_out_token, a.q_out_head = q_out_head;
    a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
    a.slots = slots;
    a.tokens = tokens;
    a.dim = (int32_t)cache->dim;
    a.q_heads = (int32_t)q_heads;
    a.wide = whole_pieces(q, q_token, q_head) && whole_pieces(q_out, q_out_token, q_out_head) && whole_pieces(k, k_token, k_head) &&
             whole_pieces(v, v_token, v_head);
    return sngguf::launch_head_rotary(a, 1, static_cast<hipStream_t>(stream));
}

int sngguf_cache_read(const sngguf_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out, void* stream) {
    const int rc = check_cache(cache);
    if (rc != SNGGUF_OK) return rc;
    // (one thread for eight elements; kv_heads and dim / 8 together below 2^21)
    if (tokens < 0 || tokens >= kMost || !launch_fits((tokens * cache->kv_heads * (cache->dim / 8) + 255) / 256, 256)) return SNGGUF_E_BADSHAPE;
    if (tokens == 0) return SNGGUF_OK;
    if (!slots || !k_out || !v_out) return SNGGUF_E_NULLPTR;
    if (!aligned(slots, 8) || !aligned(k_out, 16) || !aligned(v_out, 16)) return SNGGUF_E_ALIGN;
    RotaryCacheArgs a = {};
    set_cache(a, cache);
    a.slots = slots;
    a.tokens = tokens;
    a.dim = (int32_t)cache->dim;
    a.k_out = static_cast<bf16_t*>(k_out);
    a.v_out = static_cast<bf16_t*>(v_out);
    return sngguf::launch_cache_read(a, cache->qtype == SNGGUF_TYPE_Q8_0, static_cast<hipStream_t>(stream));
}

int64_t sngguf_attention_workspace_bytes(int64_t tokens_q, int64_t tokens_k, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (tokens_q <= 0 || tokens_q >= kMost || tokens_k < 0 || tokens_k > kMostKeys || sequences <= 0 || sequences >= kMost || !heads_fit(heads, kv_heads, dim))
        return 0;
    return plan_many(tokens_q, tokens_k, sequences, heads, kv_heads, dim).partial_bytes;
}

int sngguf_attention(const void* q, int64_t tokens_q, int64_t heads, int64_t q_token, int64_t q_head, const void* k,
                     int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, int64_t tokens_k,
                     int64_t kv_heads, int64_t dim, const int32_t* ends_q, const int32_t* ends_k, int64_t sequences, float scale,
                     int causal, int64_t window, void* out, int64_t out_token, int64_t out_head, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    if (tokens_q < 0 || tokens_q >= kMost || tokens_k < 0 || tokens_k > kMostKeys || sequences < 0 || sequences >= kMost ||
        !heads_fit(heads, kv_heads, dim) || tokens_q * (heads / kv_heads) >= kMost || window < 0 || (window && !causal) || !(scale >= 1e-30f) || scale > 1e30f ||
        k_token < 0 || k_token >= kMostStride || v_token < 0 || v_token >= kMostStride)
        return SNGGUF_E_BADSHAPE;
    if (tokens_q == 0 || sequences == 0) return SNGGUF_OK;
    if (!q || !out || !ends_q || !ends_k || (tokens_k && (!k || !v))) return SNGGUF_E_NULLPTR;
    if (!whole_pieces(q, q_token, q_head) || !whole_pieces(k, k_token, k_head) || !whole_pieces(v, v_token, v_head) ||
        !whole_pieces(out, out_token, out_head) || !aligned(ends_q, 4) || !aligned(ends_k, 4) || !aligned(workspace, 16))
        return SNGGUF_E_ALIGN;
    const int d = kernel_dim(dim);
    const Launch p = plan_many(tokens_q, tokens_k, sequences, heads, kv_heads, dim);
    if (!launch_fits(p.grid, 2 * p.rows)) return SNGGUF_E_BADSHAPE;       // (a wavefront for 32 rows)
    AttentionArgs a = {};
    a.q = static_cast<const bf16_t*>(q);
    a.k = static_cast<const bf16_t*>(k);
    a.v = static_cast<const bf16_t*>(v);
    a.out = static_cast<bf16_t*>(out);
    a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
    a.out_token = out_token, a.out_head = out_head;
    a.ends_q = ends_q;
    a.ends_k = ends_k;
    a.sequences = (int32_t)sequences;
    a.tokens_q = tokens_q;
    a.tokens_k = tokens_k;
    a.heads = (int32_t)heads;
    a.kv_heads = (int32_t)kv_heads;
    a.group = (int32_t)(heads / kv_heads);
    a.dim = (int32_t)dim;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.causal = causal != 0;
    a.window = window < kMost ? window : 0;     // (no sequence is that long, and places less the window stay within 64 bits)
    a.min_rows = 1;
    a.max_rows = (int32_t)(kMost - 1);
    float* partial = p.partial_bytes && workspace && workspace_bytes >= p.partial_bytes ? static_cast<float*>(workspace) : nullptr;
    return launch_many(a, p, d, 0, partial, static_cast<hipStream_t>(stream));
}

int64_t sngguf_paged_attention_workspace_bytes(int64_t tokens_q, int64_t sequences, int64_t max_new, int64_t max_keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    if (tokens_q <= 0 || tokens_q >= kMost || sequences <= 0 || sequences >= kMost || max_new < 0 || max_keys < 0 || max_keys > kMostKeys || !heads_fit(heads, kv_heads, dim))
        return 0;
    const PagedPlan p = paged_plan(tokens_q, sequences, max_new, max_keys, heads, kv_heads, dim);
    return (p.few ? p.a.partial_bytes : 0) + (p.many ? p.b.partial_bytes : 0);
}

int sngguf_paged_attention(const void* q, int64_t tokens_q, int64_t heads, int64_t q_token, int64_t q_head, const sngguf_kv_cache* cache,
                           const int32_t* table, int64_t table_stride, int64_t table_width, const int32_t* lens, const int32_t* ends_q,
                           int64_t sequences, int64_t max_new, float scale, int64_t window, void* out, int64_t out_token,
                           int64_t out_head, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_cache(cache);
    if (rc != SNGGUF_OK) return rc;
    if (tokens_q < 0 || tokens_q >= kMost || sequences < 0 || sequences >= kMost || !heads_fit(heads, cache->kv_heads, cache->dim) ||
        tokens_q * (heads / cache->kv_heads) >= kMost || max_new < 0 || window < 0 || !(scale >= 1e-30f) || scale > 1e30f || table_width < 0 || table_width > kMostKeys / cache->page_size ||
        (sequences > 1 && table_stride < table_width) || (!ends_q && tokens_q < sequences))
        return SNGGUF_E_BADSHAPE;
    if (tokens_q == 0 || sequences == 0) return SNGGUF_OK;
    if (!q || !out || !lens || (table_width && !table)) return SNGGUF_E_NULLPTR;
    if (!whole_pieces(q, q_token, q_head) || !whole_pieces(out, out_token, out_head) || !aligned(table, 4) || !aligned(lens, 4) ||
        !aligned(ends_q, 4) || !aligned(workspace, 16))
        return SNGGUF_E_ALIGN;
    const int64_t kv_heads = cache->kv_heads;
    const int d = kernel_dim(cache->dim);
    const bool q8 = cache->qtype == SNGGUF_TYPE_Q8_0;
    const PagedPlan p = paged_plan(tokens_q, sequences, ends_q ? max_new : 1, table_width * cache->page_size, heads, kv_heads, cache->dim);
    if ((p.few && !launch_fits(p.a.grid, 256)) || (p.many && !launch_fits(p.b.grid, 2 * p.b.rows))) return SNGGUF_E_BADSHAPE;
    AttentionArgs a = {};
    a.q = static_cast<const bf16_t*>(q);
    a.out = static_cast<bf16_t*>(out);
    a.q_token = q_token, a.q_head = q_head, a.out_token = out_token, a.out_head = out_head;
    a.k_pages = cache->k;
    a.v_pages = cache->v;
    a.k_scales = static_cast<const uint16_t*>(cache->k_scale);
    a.v_scales = static_cast<const uint16_t*>(cache->v_scale);
    a.table = table;
    a.lens = lens;
    a.table_stride = table_stride;
    a.table_width = (int32_t)table_width;
    a.pages = (int32_t)cache->pages;
    a.page_shift = log2_of(cache->page_size);
    a.ends_q = ends_q;
    a.sequences = (int32_t)sequences;
    a.tokens_q = tokens_q;
    a.heads = (int32_t)heads;
    a.kv_heads = (int32_t)kv_heads;
    a.group = (int32_t)(heads / kv_heads);
    a.dim = (int32_t)cache->dim;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.causal = 1;
    a.window = window < kMost ? window : 0;
    const int64_t need = (p.few ? p.a.partial_bytes : 0) + (p.many ? p.b.partial_bytes : 0);
    float* partial = workspace && workspace_bytes >= need ? static_cast<float*>(workspace) : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.few) {
        AttentionArgs f = a;
        f.min_rows = 1;
        f.max_rows = (int32_t)p.few_rows;
        f.partial = p.a.partial_bytes ? partial : nullptr;
        f.want = p.a.want;
        f.least = kRowsLeast;
        f.grid = f.partial ? p.a.grid : p.a.tiles;
        int r = sngguf::launch_attention_rows(f, p.a.rows, d, q8, s);
        if (r == SNGGUF_OK && f.partial) r = sngguf::launch_attention_combine(f, p.a.rows, kRowsKeys, d, p.a.tiles, p.most_rows, s);
        if (r != SNGGUF_OK) return r;
    }
    if (p.many) {
        a.min_rows = (int32_t)p.few_rows + 1;
        a.max_rows = (int32_t)(kMost - 1);
        float* rest = partial && p.b.partial_bytes ? partial + (p.few ? p.a.partial_bytes / 4 : 0) : nullptr;
        return launch_many(a, p.b, d, q8 ? 2 : 1, rest, s);
    }
    return SNGGUF_OK;
}

int64_t sngguf_shared_attention_workspace_bytes(int64_t tokens_q, int64_t sequences, int64_t groups, int64_t max_new, int64_t max_keys, int64_t heads, int64_t kv_heads,
                                                int64_t dim, int qtype) {
    if (!shared_sizes_fit(tokens_q, sequences, groups, max_new, max_keys) || !heads_fit(heads, kv_heads, dim)) return 0;
    if (shared_alone(tokens_q, sequences, max_keys, heads, kv_heads, dim))
        return sngguf_paged_attention_workspace_bytes(tokens_q, sequences, max_new, max_keys, heads, kv_heads, dim);
    return shared_plan(tokens_q, sequences, groups, max_new, max_keys, heads, kv_heads, dim, qtype == SNGGUF_TYPE_Q8_0).bytes;
}

int sngguf_shared_attention(const void* q, int64_t tokens_q, int64_t heads, int64_t q_token, int64_t q_head, const sngguf_kv_cache* cache,
                            const int32_t* table, int64_t table_stride, int64_t table_width, const int32_t* lens, const int32_t* ends_q,
                            int64_t sequences, const int32_t* groups, const int32_t* shared, int64_t group_count, int64_t max_new, float scale,
                            void* out, int64_t out_token, int64_t out_head, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_cache(cache);
    if (rc != SNGGUF_OK) return rc;
    if (tokens_q < 0 || tokens_q >= kMost || sequences < 0 || sequences >= kMost || group_count < 1 || !heads_fit(heads, cache->kv_heads, cache->dim) ||
        tokens_q * (heads / cache->kv_heads) >= kMost || max_new < 0 || !(scale >= 1e-30f) || scale > 1e30f || table_width < 0 ||
        table_width > kMostKeys / cache->page_size || (sequences > 1 && table_stride < table_width) || (!ends_q && tokens_q < sequences))
        return SNGGUF_E_BADSHAPE;
    if (tokens_q == 0 || sequences == 0) return SNGGUF_OK;
    const int64_t kv_heads = cache->kv_heads, keys = table_width * cache->page_size;
    if (!ends_q) max_new = 1;
    if (!shared_sizes_fit(tokens_q, sequences, group_count, max_new, keys)) return SNGGUF_E_BADSHAPE;
    const bool alone = shared_alone(tokens_q, sequences, keys, heads, kv_heads, cache->dim);
    if (!q || !out || !lens || (table_width && !table) || !groups || !shared || (!workspace && !alone)) return SNGGUF_E_NULLPTR;
    if (!whole_pieces(q, q_token, q_head) || !whole_pieces(out, out_token, out_head) || !aligned(table, 4) || !aligned(lens, 4) ||
        !aligned(ends_q, 4) || !aligned(groups, 4) || !aligned(shared, 4) || !aligned(workspace, 16))
        return SNGGUF_E_ALIGN;
    if (alone)
        return sngguf_paged_attention(q, tokens_q, heads, q_token, q_head, cache, table, table_stride, table_width, lens, ends_q, sequences, max_new, scale, 0, out, out_token,
                                      out_head, workspace, workspace_bytes, stream);
    const int d = kernel_dim(cache->dim);
    const bool q8 = cache->qtype == SNGGUF_TYPE_Q8_0;
    const SharedPlan p = shared_plan(tokens_q, sequences, group_count, max_new, keys, heads, kv_heads, cache->dim, q8);
    if (workspace_bytes < p.bytes || !launch_fits((tokens_q * heads + 3) / 4, 256)) return SNGGUF_E_BADSHAPE;
    for (int l = 0; l < sngguf::kSharedLaunches; l++)
        if (!launch_fits(p.launch[l].grid, l == 1 ? 256 : 2 * p.launch[l].rows)) return SNGGUF_E_BADSHAPE;
    sngguf::SharedArgs s = {};
    AttentionArgs& a = s.a;
    a.q = static_cast<const bf16_t*>(q);
    a.out = static_cast<bf16_t*>(out);
    a.q_token = q_token, a.q_head = q_head, a.out_token = out_token, a.out_head = out_head;
    a.k_pages = cache->k;
    a.v_pages = cache->v;
    a.k_scales = static_cast<const uint16_t*>(cache->k_scale);
    a.v_scales = static_cast<const uint16_t*>(cache->v_scale);
    a.table = table;
    a.lens = lens;
    a.table_stride = table_stride;
    a.table_width = (int32_t)table_width;
    a.pages = (int32_t)cache->pages;
    a.page_shift = log2_of(cache->page_size);
    a.ends_q = ends_q;
    a.sequences = (int32_t)sequences;
    a.tokens_q = tokens_q;
    a.heads = (int32_t)heads;
    a.kv_heads = (int32_t)kv_heads;
    a.group = (int32_t)(heads / kv_heads);
    a.dim = (int32_t)cache->dim;
    a.scale_log2 = scale * 1.44269504088896341f;
    uint8_t* room = static_cast<uint8_t*>(workspace);
    s.groups = groups;
    s.shared = shared;
    s.group_count = (int32_t)group_count;
    s.entries = reinterpret_cast<sngguf::AttentionEntry*>(room + p.entries);
    s.sequence_of = ends_q ? reinterpret_cast<int32_t*>(room + p.sequence_of) : nullptr;
    for (int l = 0; l < sngguf::kSharedLaunches; l++) {
        sngguf::SharedLaunch& x = s.launch[l];
        x.row_shift = log2_of(p.launch[l].rows);
        x.key_shift = log2_of(l == 1 ? kRowsKeys : kTilesKeys);
        x.max_rows = p.few_rows;
        x.want = p.launch[l].want;
        x.least = l == 1 ? kRowsLeast : l == 0 ? kCommonLeast : kTilesLeast;
        x.slots = (int32_t)(p.launch[l].grid / kv_heads);
        x.map = reinterpret_cast<sngguf::AttentionEntry*>(room + p.map[l]);
        x.partial = reinterpret_cast<float*>(room + p.partial[l]);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int r = sngguf::launch_shared_plan(s, st);
    for (int l = 0; l < sngguf::kSharedLaunches && r == SNGGUF_OK; l++) {
        if (!p.launch[l].grid) continue;
        a.map = s.launch[l].map;
        a.partial = s.launch[l].partial;
        a.grid = p.launch[l].grid;
        r = l == 1 ? sngguf::launch_attention_rows(a, p.launch[l].rows, d, q8, st)
                   : sngguf::launch_attention_tiles(a, p.launch[l].rows, many_dim(cache->dim), q8 ? 2 : 1, st);
    }
    return r == SNGGUF_OK ? sngguf::launch_shared_join(s, d, st) : r;
}

}  // extern "C"
