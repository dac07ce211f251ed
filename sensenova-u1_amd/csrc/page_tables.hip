// The tables of a step of many sequences over a paged cache, from their lengths, on the device: where each one's new tokens lie
// among the packed rows, their positions and slots, and pages for sequences that outgrow theirs.
//
// With l_i tokens before the step, n_i new ones, pages of 2^s tokens, and free pages in a ring of which those from `taken` up to `given`
// are there:
//     ends_i = n_0 + ... + n_(i-1);   has_i = ceil(l_i / 2^s);   wants_i = ceil((l_i + n_i) / 2^s) - has_i;
//     page has_i + j of sequence i is free[(taken + wants_0 + ... + wants_(i-1) + j) mod ring], as long as there are any;
//     token t with ends_i <= t < ends_(i+1):  position l_i + t - ends_i, slot page[position >> s] 2^s + position mod 2^s.
// Two prefix sums over the sequences, then each token by itself.  Little memory is moved (a few bytes a sequence, 16 a token), so
// the time is launches and latencies: one workgroup does a step of up to 1024 sequences and 4096 tokens, sums, tables and tokens; larger
// ones are two launches, whose second has a thread for each token.  Passes back to back: 256 sequences of one new token 4.6 us (as two launches
// 6.0), 16 of 128 5.3 (6.2), 16 of 256 6.9 (6.3), 16 of 500 9.5 (6.5); 37 prompts in 111000 rows 6.6.  On the device the two are level at 3000 to 3500
// rows (1000 sequences of 2 6.1 and 7.5, of 4 8.4 and 7.5), but a second launch costs a call that is not replayed 4.7 us of the host's time (11.9 and 16.6
// at every one of these sizes): so 4096.
#include "page_tables.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kFill = 256;                           // threads of a workgroup of the second launch, a token each
constexpr int kStaged = 4096;                        // sequences whose ends it keeps in LDS

// Sums that stop at `most` (below 2^31), which is all that is asked of them: so 32 bits do, and such sums may be taken in any order.
__device__ __forceinline__ uint32_t add_up_to(uint32_t x, uint32_t y, uint32_t most) { return x + y < most ? x + y : most; }

// x of the workgroup's threads in front of this one, and of all of them, added up to `most`; x is no more than that.  `part`: one for each
// wavefront, that no call before used.  (In a wavefront: row shifts, then a row's last value handed on.)
__device__ __forceinline__ uint32_t block_sum_before(uint32_t x, uint32_t most, uint32_t* part, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#define SNGGUF_STEP(CONTROL, ROWS) x = add_up_to(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CONTROL, ROWS, 0xF, false), most);
    SNGGUF_STEP(0x111, 0xF)
    SNGGUF_STEP(0x112, 0xF)
    SNGGUF_STEP(0x114, 0xF)
    SNGGUF_STEP(0x118, 0xF)
    SNGGUF_STEP(0x142, 0xA)
    SNGGUF_STEP(0x143, 0xC)
#undef SNGGUF_STEP
    if (lane == 63) part[wave] = x;
    const uint32_t in_wave = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x138, 0xF, 0xF, false);      // the lane before's
    __syncthreads();
    total = 0;
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        if (w == wave) before = total;
        total = add_up_to(total, part[w], most);
    }
    return add_up_to(before, in_wave, most);
}

__device__ __forceinline__ int32_t clamped(int64_t x, int64_t lo, int64_t hi) { return (int32_t)(x < lo ? lo : x > hi ? hi : x); }
__device__ __forceinline__ int32_t pages_of(int64_t tokens, int shift) { return (int32_t)((tokens + ((int64_t)1 << shift) - 1) >> shift); }

// What the ring holds: pages that are there, and the place of the first
__device__ __forceinline__ int32_t ring_count(const PageArgs& a) { return clamped(a.cursor[1] - a.cursor[0], 0, a.ring); }
__device__ __forceinline__ int32_t ring_place(int64_t at, int32_t ring) {
    if ((at >> 32) == 0) return (int32_t)((uint32_t)at % (uint32_t)ring);
    const int64_t r = at % ring;
    return (int32_t)(r < 0 ? r + ring : r);
}
__device__ __forceinline__ int32_t ring_step(int32_t at, int64_t by, int32_t ring) {      // 0 <= by <= ring
    const int64_t r = at + by;
    return (int32_t)(r >= ring ? r - ring : r);
}

// Sequence of token t: the one whose end is the first behind it (those without new tokens end where they start); ends[0] is 0
__device__ __forceinline__ int32_t sequence_of(const int32_t* ends, int32_t sequences, int32_t t) {
    int32_t lo = 0, hi = sequences;                  // ends[lo] <= t < ends[hi]
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (ends[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void fill_token(const PageArgs& a, int64_t t, int32_t i, int32_t end, const PageSequence& q) {
    const int64_t position = (int64_t)q.length + (t - end);
    int64_t slot = -1;
    if (position < q.after) {
        const int32_t column = (int32_t)(position >> a.page_shift);
        int32_t* row = a.pages + (int64_t)i * a.width;
        int32_t page;
        if (column < q.pages) {
            page = row[column];
        } else {
            page = a.free[ring_step(q.ring_at, column - q.pages, a.ring)];
            // (every page that a sequence gets has its first token among the new ones)
            if ((position & ((1 << a.page_shift) - 1)) == 0) row[column] = page;
        }
        slot = ((int64_t)page << a.page_shift) + (position & ((1 << a.page_shift) - 1));
    }
    a.positions[t] = position;
    a.slots[t] = slot;
}

}  // namespace

template <bool ONE>
__global__ __launch_bounds__(kThreads) void page_append_kernel(PageArgs a) {
    __shared__ uint32_t part[2][2][kWaves];
    __shared__ unsigned long long missing;
    __shared__ int32_t ends[ONE ? kOneLaunchSequences + 1 : 1];
    __shared__ PageSequence of[ONE ? kOneLaunchSequences : 1];
    touch_arguments(a);
    const int tid = threadIdx.x;
    const int64_t most = (int64_t)a.width << a.page_shift;
    const int64_t taken = a.cursor[0], given = a.cursor[1];
    const int32_t there = ring_count(a), first = ring_place(taken, a.ring);
    const uint32_t room_rows = (uint32_t)a.tokens, room_pages = 0x7FFFFFFFu;
    uint32_t rows = 0, wanted = 0;
    if (tid == 0) {
        a.ends[0] = 0;
        missing = 0;
        if constexpr (ONE) ends[0] = 0;
    }
    for (int64_t base = 0; base < a.sequences; base += kThreads) {
        const int64_t i = base + tid;
        const bool mine = i < a.sequences;
        const int turn = (base / kThreads) & 1;
        const int32_t asked = mine ? a.added[i] : 0;
        const int32_t length = mine ? clamped(a.lens[i], 0, most) : 0;
        // (more new tokens than there are rows: those behind the last row are none)
        const uint32_t n = asked < 0 ? 0 : (uint32_t)asked < room_rows ? (uint32_t)asked : room_rows;
        uint32_t sum;
        const uint32_t e0 = add_up_to(rows, block_sum_before(n, room_rows, part[turn][0], sum), room_rows), e1 = add_up_to(e0, n, room_rows);
        rows = add_up_to(rows, sum, room_rows);
        const int64_t whole = length + (int64_t)(e1 - e0);
        const int32_t has = pages_of(length, a.page_shift), wants = pages_of(whole < most ? whole : most, a.page_shift) - has;
        const uint32_t before = add_up_to(wanted, block_sum_before((uint32_t)wants, room_pages, part[turn][1], sum), room_pages);
        wanted = add_up_to(wanted, sum, room_pages);
        const int32_t gets = clamped((int64_t)there - before, 0, wants);
        const int64_t room = (int64_t)(has + gets) << a.page_shift;
        PageSequence q;
        q.length = length;
        q.after = (int32_t)(whole < room ? whole : room);
        q.pages = has;
        q.ring_at = gets ? ring_step(first, before, a.ring) : 0;
        if (whole > q.after) atomicAdd(&missing, (unsigned long long)(whole - q.after));
        if (mine) {
            a.ends[i + 1] = (int32_t)e1;
            a.lens_out[i] = q.after;
            if constexpr (ONE) ends[i + 1] = (int32_t)e1, of[i] = q;
            else a.of[i] = q;
        }
    }
    __syncthreads();
    if (tid == 0) {
        *a.missing = missing < 0x7FFFFFFFull ? (int32_t)missing : 0x7FFFFFFF;
        a.cursor_out[0] = taken + (wanted < (uint32_t)there ? wanted : there);
        a.cursor_out[1] = given;
    }
    if constexpr (ONE) {
        const int32_t total = (int32_t)rows;
        for (int64_t t = tid; t < a.tokens; t += kThreads) {
            if (t < total) {
                const int32_t i = sequence_of(ends, (int32_t)a.sequences, (int32_t)t);
                fill_token(a, t, i, ends[i], of[i]);
            } else {
                a.positions[t] = 0;
                a.slots[t] = -1;
            }
        }
    }
}

__global__ __launch_bounds__(kFill) void page_fill_kernel(PageArgs a) {
    __shared__ int32_t staged[kStaged + 1];
    const bool stage = a.sequences <= kStaged;
    if (stage) {
        for (int i = threadIdx.x; i <= a.sequences; i += kFill) staged[i] = a.ends[i];
        __syncthreads();
    }
    const int32_t* ends = stage ? staged : a.ends;
    const int32_t total = ends[a.sequences];
    const int64_t t = (int64_t)blockIdx.x * kFill + threadIdx.x;
    if (t >= a.tokens) return;
    if (t < total) {
        const int32_t i = sequence_of(ends, (int32_t)a.sequences, (int32_t)t);
        fill_token(a, t, i, ends[i], a.of[i]);
    } else {
        a.positions[t] = 0;
        a.slots[t] = -1;
    }
}

// Pages of the sequences that are done back into the ring, in the order of the sequences; a wavefront copies one's.
__global__ __launch_bounds__(kThreads) void page_release_kernel(PageArgs a) {
    __shared__ uint32_t part[kWaves];
    __shared__ int32_t offset[kThreads], from[kThreads], count[kThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t most = (int64_t)a.width << a.page_shift;
    const int64_t given = a.cursor[1];
    const int32_t room = a.ring - ring_count(a), first = ring_place(given, a.ring);
    const uint32_t all = 0x7FFFFFFFu;
    uint32_t back = 0;
    for (int64_t base = 0; base < a.sequences; base += kThreads) {
        const int64_t i = base + tid;
        const bool done = i < a.sequences && a.done[i];
        const int32_t has = done ? pages_of(clamped(a.lens[i], 0, most), a.page_shift) : 0;
        const int32_t held = done && a.held ? clamped(a.held[i], 0, has) : 0;
        uint32_t sum;
        offset[tid] = (int32_t)add_up_to(back, block_sum_before((uint32_t)(has - held), all, part, sum), all);
        from[tid] = held;
        count[tid] = has - held;
        back = add_up_to(back, sum, all);
        __syncthreads();
        for (int k = wave; k < kThreads && base + k < a.sequences; k += kWaves) {
            const int32_t* row = a.pages + (base + k) * a.width + from[k];
            for (int32_t j = lane; j < count[k] && j < (int64_t)room - offset[k]; j += 64) a.free[ring_step(first, (int64_t)offset[k] + j, a.ring)] = row[j];
        }
        if (done) {
            a.lens[i] = 0;
            if (a.held) a.held[i] = 0;
        }
        __syncthreads();
    }
    if (tid == 0) a.cursor[1] = given + (back < (uint32_t)room ? back : room);
}

// A workgroup a sequence: one that is empty starts with whole pages of its parent, which stay the parent's.
__global__ __launch_bounds__(kFill) void page_fork_kernel(PageArgs a) {
    const int64_t i = blockIdx.x;
    const int32_t p = a.parent[i];
    if (p < 0 || p >= a.sequences || p == i || a.parent[p] >= 0) return;
    const int32_t length = a.lens[i];
    const int32_t has = clamped(a.lens[p], 0, (int64_t)a.width << a.page_shift), common = a.common[i];
    const int32_t pages = (common < has ? common < 0 ? 0 : common : has) >> a.page_shift;
    __syncthreads();
    if (length != 0) return;
    for (int32_t j = threadIdx.x; j < pages; j += kFill) a.pages[i * a.width + j] = a.pages[(int64_t)p * a.width + j];
    if (threadIdx.x == 0) {
        a.lens[i] = pages << a.page_shift;
        a.held[i] = pages;
    }
}

int launch_page_append(const PageArgs& a, bool one, hipStream_t stream) {
    if (one) {
        page_append_kernel<true><<<1, kThreads, 0, stream>>>(a);
    } else {
        page_append_kernel<false><<<1, kThreads, 0, stream>>>(a);
        if (hipGetLastError() != hipSuccess) return SNGGUF_E_LAUNCH;      // (asking clears it)
        if (a.tokens) page_fill_kernel<<<dim3((unsigned)((a.tokens + kFill - 1) / kFill)), kFill, 0, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

int launch_page_release(const PageArgs& a, hipStream_t stream) {
    page_release_kernel<<<1, kThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

int launch_page_fork(const PageArgs& a, hipStream_t stream) {
    page_fork_kernel<<<dim3((unsigned)a.sequences), kFill, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

}  // namespace sngguf
