// Copies inside the cache: pages that several sequences share and one of them is about to write (the first positions of each, of
// every cache entry, keys and values), and states of fixed size for sequences that continue the same one.
//
// A move is (source, destination, positions).  Moves of one source are one group: its bytes are read once and stored to every
// destination, so a call moves what it cannot do without: each source in, each destination out.  The list of moves
// travels as the kernel's argument (no buffer, no copy to the device); a call of more moves than an argument holds is
// several launches.  Sources are never destinations and no destination comes twice (the caller sees to it), so the order of
// CTAs does not matter.
//
// Pages: a CTA takes a head of an entry of one source.  Its keys are one run of bytes (positions follow one another), its values head_dim rows of
// 64 positions of which the first n are taken; 16 bytes an access, two of the keys, two of the values and two of the values' ends a thread asked
// for before the first is stored (four of each take 96 registers, half the CTAs, and are no faster).  States: a CTA takes 2,048 accesses (of the
// widest that the addresses allow) of one state, eight a thread.
//
// Bound by HBM, and where pages are not full by the sectors that rows of values end in: they are read to be written.  Measured: 40 pages of
// 1 to 64 positions in 32 layers of 8 heads of 128, bfloat16, 81 us: 449 MB move (5.6 TB/s) where 260 MB are asked for; pages filled to a
// multiple of 16 positions run at 5 to 6.3 TB/s of what is asked for.  19 states of 2.4 MB to 37
// places, 134 MB, 23.5 us, 5.7 TB/s.
#include "common.cuh"

namespace b200 {

constexpr int kCopyThreads = 256;
constexpr int kPageAtOnce = 2, kTailAtOnce = 2, kSlotAtOnce = 8;
constexpr int kMaxSources = 96, kMaxDestinations = 256;     // of one launch (an argument holds 4 KB)

struct Moves {
    int source[kMaxSources], positions[kMaxSources], first[kMaxSources + 1], destination[kMaxDestinations];
};

struct Pages {
    unsigned char* keys;
    unsigned char* values;
    long long entry, page;      // bytes between entries and between pages
    int head, kv_heads;         // bytes of a head's keys or values, heads
    int head_dim, element;
};

// the first `bytes` (even, at most 16) of `w`, the others of `old`
__device__ __forceinline__ uint4 blended(const uint4& w, const uint4& old, int bytes) {
    const unsigned a[4] = {w.x, w.y, w.z, w.w}, b[4] = {old.x, old.y, old.z, old.w};
    unsigned r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = bytes - 4 * i;
        r[i] = left >= 4 ? a[i] : left == 2 ? (a[i] & 0xffffu) | (b[i] & 0xffff0000u) : b[i];
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

__global__ void __launch_bounds__(kCopyThreads, 4) copy_pages_kernel(const __grid_constant__ Moves moves, const __grid_constant__ Pages p) {
    pdl_launch_dependents();
    pdl_wait();
    const int group = blockIdx.y, entry = blockIdx.x / p.kv_heads, head = blockIdx.x - entry * p.kv_heads, positions = moves.positions[group];
    const size_t at = (size_t)entry * p.entry + (size_t)head * p.head;
    const int row_bytes = positions * p.element, pitch = kPageTokens * p.element, first = moves.first[group], last = moves.first[group + 1];
    const unsigned char* from_k = p.keys + at + (size_t)moves.source[group] * p.page;
    const unsigned char* from_v = p.values + at + (size_t)moves.source[group] * p.page;
    // What a row of values has in its last sector, if that is not full.  The sector is stored whole, with what the destination has behind the last
    // position: a store of a part of a sector costs HBM a read and a write of its own (40 pages of 31 positions took 103 us, of 32 53 us).
    const int tail = row_bytes % 32, tail_at = row_bytes - tail, n_tails = tail ? (last - first) * p.head_dim * 2 : 0;
    uint4 old[kTailAtOnce], fresh[kTailAtOnce];
    auto tail_place = [&](int i) {          // piece i of the tails: destinations, rows, two halves
        const int d = i / (2 * p.head_dim), r = i - d * 2 * p.head_dim;
        return make_int2(first + d, (r >> 1) * pitch + tail_at + (r & 1) * 16);
    };
    auto ask_tails = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kTailAtOnce; ++u) {
            const int i = i0 + u * kCopyThreads;
            if (i >= n_tails) continue;
            const int2 t = tail_place(i);
            old[u] = *reinterpret_cast<const uint4*>(p.values + at + (size_t)moves.destination[t.x] * p.page + t.y);
            fresh[u] = *reinterpret_cast<const uint4*>(from_v + t.y);
        }
    };
    ask_tails(threadIdx.x);
    const int n_keys = positions * p.head_dim * p.element / 16;                     // (a position's keys are whole pieces)
    const int per = row_bytes / 32 * 2, n_values = per * p.head_dim;
    const unsigned magic = per > 0 ? (unsigned)(((1ull << 32) + per - 1) / per) : 0u;   // (exact: pieces are below 2^16, per is 2 to 16)
    for (int i0 = threadIdx.x; i0 < max(n_keys, n_values); i0 += kCopyThreads * kPageAtOnce) {
        uint4 k[kPageAtOnce], v[kPageAtOnce];
        int place[kPageAtOnce];
#pragma unroll
        for (int u = 0; u < kPageAtOnce; ++u) {
            const int i = i0 + u * kCopyThreads, row = (int)__umulhi((unsigned)i, magic);
            place[u] = row * pitch + (i - row * per) * 16;
            if (i < n_keys) k[u] = *reinterpret_cast<const uint4*>(from_k + i * 16);
            if (i < n_values) v[u] = *reinterpret_cast<const uint4*>(from_v + place[u]);
        }
        for (int d = first; d < last; ++d) {
            const size_t to = at + (size_t)moves.destination[d] * p.page;
#pragma unroll
            for (int u = 0; u < kPageAtOnce; ++u) {
                const int i = i0 + u * kCopyThreads;
                if (i < n_keys) *reinterpret_cast<uint4*>(p.keys + to + i * 16) = k[u];
                if (i < n_values) *reinterpret_cast<uint4*>(p.values + to + place[u]) = v[u];
            }
        }
    }
    for (int i0 = threadIdx.x; i0 < n_tails; i0 += kCopyThreads * kTailAtOnce) {
        if (i0 >= kCopyThreads * kTailAtOnce) ask_tails(i0);
#pragma unroll
        for (int u = 0; u < kTailAtOnce; ++u) {
            const int i = i0 + u * kCopyThreads;
            if (i >= n_tails) continue;
            const int2 t = tail_place(i);
            *reinterpret_cast<uint4*>(p.values + at + (size_t)moves.destination[t.x] * p.page + t.y) =
                blended(fresh[u], old[u], min(16, max(0, tail - (i & 1) * 16)));
        }
    }
}

struct Slots {
    unsigned char* data;
    long long entry, slot, pieces;      // bytes between entries and between slots; accesses of a state
    int blocks;                         // CTAs of a state
};

template <typename W>
__global__ void __launch_bounds__(kCopyThreads) copy_slots_kernel(const __grid_constant__ Moves moves, const __grid_constant__ Slots s) {
    pdl_launch_dependents();
    pdl_wait();
    const int entry = blockIdx.x / s.blocks, block = blockIdx.x - entry * s.blocks, group = blockIdx.y;
    const long long i0 = (long long)block * (kCopyThreads * kSlotAtOnce) + threadIdx.x;
    unsigned char* at = s.data + (size_t)entry * s.entry;
    const W* from = reinterpret_cast<const W*>(at + (size_t)moves.source[group] * s.slot) + i0;
    W v[kSlotAtOnce];
#pragma unroll
    for (int u = 0; u < kSlotAtOnce; ++u) if (i0 + u * kCopyThreads < s.pieces) v[u] = from[u * kCopyThreads];
    for (int d = moves.first[group]; d < moves.first[group + 1]; ++d) {
        W* to = reinterpret_cast<W*>(at + (size_t)moves.destination[d] * s.slot) + i0;
#pragma unroll
        for (int u = 0; u < kSlotAtOnce; ++u) if (i0 + u * kCopyThreads < s.pieces) to[u * kCopyThreads] = v[u];
    }
}

// As many launches as the lists need: `launch(moves, number of sources)` each.
template <typename Launch>
static int in_arguments(const int* sources, const int* positions, const int* firsts, int n_sources, const int* destinations, Launch launch) {
    Moves m;
    int at = 0, done = 0;       // source and destination reached
    while (at < n_sources) {
        int n = 0, count = 0;
        while (at < n_sources && n < kMaxSources && count < kMaxDestinations) {
            const int left = firsts[at + 1] - done, room = kMaxDestinations - count, take = left < room ? left : room;
            m.source[n] = sources[at];
            m.positions[n] = positions ? positions[at] : 0;
            m.first[n] = count;
            for (int i = 0; i < take; ++i) m.destination[count + i] = destinations[done + i];
            count += take;
            done += take;
            ++n;
            if (done == firsts[at + 1]) ++at;
        }
        m.first[n] = count;
        const int st = launch(m, n);
        if (st != 0) return st;
    }
    return 0;
}

}  // namespace b200

// Host lists: n_sources sources with the positions to take of each, and firsts[i] .. firsts[i + 1] of the destinations for source i
// (firsts[0] = 0).  keys [entry][page][kv_head][64][head_dim], values [entry][page][kv_head][head_dim][64], entries `entry_elements`
// elements apart, `element` bytes each (2 or 4).
extern "C" int b200_copy_pages(void* keys, void* values, long long entry_elements, int n_entries, int n_kv_heads, int head_dim, int element,
                               const int* sources, const int* positions, const int* firsts, int n_sources, const int* destinations,
                               cudaStream_t stream) {
    using namespace b200;
    if (n_sources <= 0 || n_entries <= 0) return 0;
    if (n_kv_heads < 1 || head_dim < 1 || (element != 2 && element != 4)) return kErrBadArgument;
    if ((head_dim * element) % 16 != 0 || (entry_elements * element) % 16 != 0 || (((uintptr_t)keys | (uintptr_t)values) & 15) != 0)
        return kErrUnsupportedSize;
    if ((long long)n_entries * n_kv_heads > 0x7fffffffll || head_dim > 1024) return kErrUnsupportedSize;
    const long long head = (long long)kPageTokens * head_dim * element;
    const Pages p{(unsigned char*)keys, (unsigned char*)values, entry_elements * element, head * n_kv_heads, (int)head, n_kv_heads, head_dim, element};
    return in_arguments(sources, positions, firsts, n_sources, destinations, [&](const Moves& m, int n) {
        return launch_pdl(copy_pages_kernel, dim3(n_entries * n_kv_heads, n), dim3(kCopyThreads), 0, stream, m, p);
    });
}

// data [entry][slot] of `bytes` bytes each, slots `slot_stride` bytes apart, entries `entry_stride`; lists as above, without positions.
extern "C" int b200_copy_slots(void* data, long long entry_stride, long long slot_stride, long long bytes, int n_entries, const int* sources,
                               const int* firsts, int n_sources, const int* destinations, cudaStream_t stream) {
    using namespace b200;
    if (n_sources <= 0 || n_entries <= 0 || bytes <= 0) return 0;
    const unsigned long long all = (unsigned long long)(uintptr_t)data | entry_stride | slot_stride | bytes;
    int width = 16;
    while (all % width) width /= 2;
    const long long pieces = bytes / width, blocks = (pieces + kCopyThreads * kSlotAtOnce - 1) / (kCopyThreads * kSlotAtOnce);
    if (blocks * n_entries > 0x7fffffffll) return kErrUnsupportedSize;
    const Slots s{(unsigned char*)data, entry_stride, slot_stride, pieces, (int)blocks};
    return in_arguments(sources, nullptr, firsts, n_sources, destinations, [&](const Moves& m, int n) {
        const dim3 grid((unsigned)(blocks * n_entries), n), block(kCopyThreads);
        switch (width) {
            case 16: return launch_pdl(copy_slots_kernel<uint4>, grid, block, 0, stream, m, s);
            case 8: return launch_pdl(copy_slots_kernel<uint2>, grid, block, 0, stream, m, s);
            case 4: return launch_pdl(copy_slots_kernel<unsigned int>, grid, block, 0, stream, m, s);
            case 2: return launch_pdl(copy_slots_kernel<unsigned short>, grid, block, 0, stream, m, s);
            default: return launch_pdl(copy_slots_kernel<unsigned char>, grid, block, 0, stream, m, s);
        }
    });
}
