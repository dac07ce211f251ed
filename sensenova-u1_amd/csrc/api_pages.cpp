// extern "C" entry points of the page tables of many sequences.  Argument checks and the choice of kernels; nothing here
// allocates, synchronises or throws.
#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "page_tables.hpp"

namespace {

using sngguf::PageArgs;

constexpr int64_t kMost = (int64_t)1 << 31;
constexpr int64_t kMostKeys = kMost - 65536;          // tokens of a sequence
constexpr int64_t kMostSequences = (int64_t)1 << 24;  // a workgroup of 256 threads each, threads numbered with 32 bits

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Bytes {
    const void* at;
    int64_t count;
};
bool overlap(const Bytes& x, const Bytes& y) {
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x.at), y0 = reinterpret_cast<uintptr_t>(y.at);
    return x.at && y.at && x.count && y.count && x0 < y0 + (uintptr_t)y.count && y0 < x0 + (uintptr_t)x.count;
}
// Whether `x` shares no byte with any of them
template <int N>
bool apart(const Bytes& x, const Bytes (&others)[N]) {
    for (const Bytes& y : others)
        if (overlap(x, y)) return false;
    return true;
}

// Whether the tables' arrays share no byte (a call writes some while others of its threads still read)
bool tables_apart(const PageArgs& a) {
    const Bytes pages = {a.pages, a.sequences * a.width * 4}, lens = {a.lens, a.sequences * 4}, held = {a.held, a.sequences * 4}, free = {a.free, (int64_t)a.ring * 4}, cursor = {a.cursor, 16};
    const Bytes behind_pages[] = {lens, held, free, cursor}, behind_lens[] = {held, free, cursor}, behind_held[] = {free, cursor}, behind_free[] = {cursor};
    return apart(pages, behind_pages) && apart(lens, behind_lens) && apart(held, behind_held) && apart(free, behind_free);
}

int check_tables(const sngguf_page_tables* t, PageArgs& a) {
    if (!t) return SNGGUF_E_NULLPTR;
    if (t->sequences < 0 || t->sequences >= kMostSequences || t->width < 1 || t->ring < 1 || t->ring >= kMost || t->page_size < 16 || t->page_size > 4096 ||
        (t->page_size & (t->page_size - 1)) != 0 || t->width > kMostKeys / t->page_size)
        return SNGGUF_E_BADSHAPE;
    if (t->sequences == 0) return SNGGUF_OK;
    if (!t->pages || !t->lens || !t->free || !t->cursor) return SNGGUF_E_NULLPTR;
    if (!aligned(t->pages, 4) || !aligned(t->lens, 4) || !aligned(t->held, 4) || !aligned(t->free, 4) || !aligned(t->cursor, 8)) return SNGGUF_E_ALIGN;
    a.pages = t->pages;
    a.lens = t->lens;
    a.held = t->held;
    a.free = t->free;
    a.cursor = t->cursor;
    a.sequences = t->sequences;
    a.width = (int32_t)t->width;
    a.ring = (int32_t)t->ring;
    while (((int64_t)1 << a.page_shift) < t->page_size) a.page_shift++;
    return SNGGUF_OK;
}

bool one_launch(int64_t sequences, int64_t tokens) { return sequences <= sngguf::kOneLaunchSequences && tokens <= sngguf::kOneLaunchTokens; }

}  // namespace

extern "C" {

int64_t sngguf_page_append_workspace_bytes(int64_t sequences, int64_t tokens) {
    if (sequences <= 0 || sequences >= kMostSequences || tokens < 0 || tokens >= kMost || one_launch(sequences, tokens)) return 0;
    return sequences * (int64_t)sizeof(sngguf::PageSequence);
}

int sngguf_page_append(const sngguf_page_tables* tables, const int32_t* added, int64_t tokens, int32_t* ends, int32_t* lens_out, int64_t* cursor_out,
                       int64_t* positions, int64_t* slots, int32_t* missing, void* workspace, int64_t workspace_bytes, void* stream) {
    PageArgs a = {};
    const int rc = check_tables(tables, a);
    if (rc != SNGGUF_OK) return rc;
    if (tokens < 0 || tokens >= kMost) return SNGGUF_E_BADSHAPE;
    if (a.sequences == 0) return SNGGUF_OK;
    const int64_t need = sngguf_page_append_workspace_bytes(a.sequences, tokens);
    if (!added || !ends || !lens_out || !cursor_out || !missing || (tokens && (!positions || !slots)) || (need && !workspace)) return SNGGUF_E_NULLPTR;
    if (need && workspace_bytes < need) return SNGGUF_E_BADSHAPE;
    if (!aligned(added, 4) || !aligned(ends, 4) || !aligned(lens_out, 4) || !aligned(cursor_out, 8) || !aligned(positions, 8) || !aligned(slots, 8) ||
        !aligned(missing, 4) || !aligned(workspace, 16))
        return SNGGUF_E_ALIGN;
    // What is written, the tables' lengths and cursor among it where they are given for it, and nothing else in part
    const Bytes written[] = {{lens_out, a.sequences * 4}, {cursor_out, 16}, {ends, (a.sequences + 1) * 4}, {missing, 4}, {positions, tokens * 8}, {slots, tokens * 8}, {workspace, need}};
    const Bytes tables_of[] = {{a.pages, a.sequences * a.width * 4}, {a.held, a.sequences * 4}, {a.free, (int64_t)a.ring * 4}, {a.lens, a.sequences * 4}, {a.cursor, 16}};
    if (!tables_apart(a) || !apart({added, a.sequences * 4}, written) || overlap({added, a.sequences * 4}, tables_of[0])) return SNGGUF_E_BADSHAPE;
    for (const Bytes& x : written) {
        for (const Bytes& y : written)
            if (&x != &y && overlap(x, y)) return SNGGUF_E_BADSHAPE;
        for (const Bytes& y : tables_of)
            if (overlap(x, y) && !(x.at == y.at && ((x.at == lens_out && y.at == a.lens) || (x.at == cursor_out && y.at == a.cursor)))) return SNGGUF_E_BADSHAPE;
    }
    a.added = added;
    a.tokens = tokens;
    a.ends = ends;
    a.lens_out = lens_out;
    a.cursor_out = cursor_out;
    a.positions = positions;
    a.slots = slots;
    a.missing = missing;
    a.of = static_cast<sngguf::PageSequence*>(workspace);
    return sngguf::launch_page_append(a, need == 0, static_cast<hipStream_t>(stream));
}

int sngguf_page_release(const sngguf_page_tables* tables, const uint8_t* done, void* stream) {
    PageArgs a = {};
    const int rc = check_tables(tables, a);
    if (rc != SNGGUF_OK || a.sequences == 0) return rc;
    if (!done) return SNGGUF_E_NULLPTR;
    const Bytes written[] = {{a.lens, a.sequences * 4}, {a.held, a.sequences * 4}, {a.free, (int64_t)a.ring * 4}, {a.cursor, 16}};
    if (!tables_apart(a) || !apart({done, a.sequences}, written)) return SNGGUF_E_BADSHAPE;
    a.done = done;
    return sngguf::launch_page_release(a, static_cast<hipStream_t>(stream));
}

int sngguf_page_fork(const sngguf_page_tables* tables, const int32_t* parent, const int32_t* common, void* stream) {
    PageArgs a = {};
    const int rc = check_tables(tables, a);
    if (rc != SNGGUF_OK || a.sequences == 0) return rc;
    if (!parent || !common || !a.held) return SNGGUF_E_NULLPTR;
    if (!aligned(parent, 4) || !aligned(common, 4)) return SNGGUF_E_ALIGN;
    const Bytes written[] = {{a.pages, a.sequences * a.width * 4}, {a.lens, a.sequences * 4}, {a.held, a.sequences * 4}};
    if (!tables_apart(a) || !apart({parent, a.sequences * 4}, written) || !apart({common, a.sequences * 4}, written)) return SNGGUF_E_BADSHAPE;
    a.parent = parent;
    a.common = common;
    return sngguf::launch_page_fork(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
