// Copies inside the cache: pages that several sequences share and one of them is about to write (the first positions of each, of
// every cache entry, keys and values), and states of fixed size for sequences that continue the same one.
//
// A move is (source, destination, positions).  Moves of one source are one group: its bytes are read once and stored to every
// destination, so a call moves what it cannot do without: each source in, each destination out.  The list of moves
// travels as the kernel's argument (no buffer, no copy to the device); a call of more moves than an argument holds is
// several launches.  Sources are never destinations and no destination comes twice (the caller sees to it), so the order of
// CTAs does not matter.
//
// What is copied lies in slabs: of a page and entry, a head's keys are one run of bytes (positions are rows), its values are
// head_dim rows of 64 positions of which the first n are taken; a state is cut into runs of 16 KB.  A CTA takes one slab of one
// source, four 16-byte loads a thread at a time.  Bound by HBM.
#include "common.cuh"

namespace b200 {

constexpr int kCopyThreads = 128;
constexpr int kCopyAtOnce = 4;
constexpr int kMaxSources = 96, kMaxDestinations = 256;     // of one launch (an argument holds 4 KB)
constexpr int kStateSlab = 16384;

struct Moves {
    int source[kMaxSources], positions[kMaxSources], first[kMaxSources + 1], destination[kMaxDestinations];
};

struct Slabs {              // a kind of storage: [entry][index][slab of rows]
    unsigned char* base;
    long long entry_stride, index_stride, slab_stride, row_stride;      // bytes
    long long bytes;        // of an index and entry (states: the last slab is cut there); 0: slabs are whole
    int per_index;          // slabs of an index and entry
    int rows;               // of a slab
    int position_bytes;     // of a row and position
};

// W: bytes of an access.  What remains of a row behind its whole accesses is blended into the destination's bytes.
template <typename W>
__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const __grid_constant__ Moves moves, const __grid_constant__ Slabs a,
                                                                 const __grid_constant__ Slabs b, int slabs_a) {
    pdl_launch_dependents();
    pdl_wait();
    const bool second = (int)blockIdx.x >= slabs_a;
    const Slabs& s = second ? b : a;
    const int at = second ? blockIdx.x - slabs_a : blockIdx.x;
    const int entry = at / s.per_index, slab = at % s.per_index;
    const int group = blockIdx.y;
    const size_t offset = (size_t)entry * s.entry_stride + (size_t)slab * s.slab_stride;
    const unsigned char* from = s.base + offset + (size_t)moves.source[group] * s.index_stride;
    long long row_bytes = (long long)moves.positions[group] * s.position_bytes;
    if (s.bytes) row_bytes = min(row_bytes, s.bytes - (long long)slab * s.slab_stride);
    const int per_row = (int)((row_bytes + sizeof(W) - 1) / sizeof(W)), n = per_row * s.rows;
    const int rest = (int)(row_bytes % sizeof(W));       // bytes of a row's last access, if it is not whole
    const int first = moves.first[group], last = moves.first[group + 1];
    for (int i0 = threadIdx.x; i0 < n; i0 += kCopyThreads * kCopyAtOnce) {
        W v[kCopyAtOnce];
        size_t where[kCopyAtOnce];
        bool cut[kCopyAtOnce];
#pragma unroll
        for (int u = 0; u < kCopyAtOnce; ++u) {
            const int i = i0 + u * kCopyThreads, row = i / per_row, c = i - row * per_row;
            where[u] = (size_t)row * s.row_stride + (size_t)c * sizeof(W);
            cut[u] = rest != 0 && c == per_row - 1;
            if (i < n) v[u] = *reinterpret_cast<const W*>(from + where[u]);
        }
        for (int d = first; d < last; ++d) {
            unsigned char* to = s.base + offset + (size_t)moves.destination[d] * s.index_stride;
#pragma unroll
            for (int u = 0; u < kCopyAtOnce; ++u) {
                if (i0 + u * kCopyThreads >= n) continue;
                if (!cut[u]) {
                    *reinterpret_cast<W*>(to + where[u]) = v[u];
                } else {        // (elements are of two bytes or four: so is what remains)
                    const unsigned short* halves = reinterpret_cast<const unsigned short*>(&v[u]);
#pragma unroll
                    for (int k = 0; k < (int)sizeof(W) / 2; ++k)
                        if (2 * k < rest) reinterpret_cast<unsigned short*>(to + where[u])[k] = halves[k];
                }
            }
        }
    }
}

static int launch_copies(const int* sources, const int* positions, const int* firsts, int n_sources, const int* destinations, const Slabs& a,
                         const Slabs& b, int slabs_a, int slabs_b, int width, cudaStream_t stream) {
    Moves m;
    int at = 0, done = 0;       // source and destination reached
    while (at < n_sources) {
        int n = 0, count = 0;
        while (at < n_sources && n < kMaxSources && count < kMaxDestinations) {
            const int take = min(firsts[at + 1] - done, kMaxDestinations - count);
            m.source[n] = sources[at];
            m.positions[n] = positions ? positions[at] : 1;     // (a state's slab is its one position)
            m.first[n] = count;
            for (int i = 0; i < take; ++i) m.destination[count + i] = destinations[done + i];
            count += take;
            done += take;
            ++n;
            if (done == firsts[at + 1]) ++at;
        }
        m.first[n] = count;
        const dim3 grid(slabs_a + slabs_b, n), block(kCopyThreads);
        int st;
        switch (width) {
            case 16: st = launch_pdl(cache_copy_kernel<uint4>, grid, block, 0, stream, m, a, b, slabs_a); break;
            case 8: st = launch_pdl(cache_copy_kernel<uint2>, grid, block, 0, stream, m, a, b, slabs_a); break;
            case 4: st = launch_pdl(cache_copy_kernel<unsigned int>, grid, block, 0, stream, m, a, b, slabs_a); break;
            case 2: st = launch_pdl(cache_copy_kernel<unsigned short>, grid, block, 0, stream, m, a, b, slabs_a); break;
            default: st = launch_pdl(cache_copy_kernel<unsigned char>, grid, block, 0, stream, m, a, b, slabs_a); break;
        }
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
    const long long head = (long long)kPageTokens * head_dim * element, page = head * n_kv_heads, entry = entry_elements * element;
    const Slabs k{(unsigned char*)keys, entry, page, head, head, 0, n_kv_heads, 1, head_dim * element};
    const Slabs v{(unsigned char*)values, entry, page, head, kPageTokens * element, 0, n_kv_heads, head_dim, element};
    const int slabs = n_entries * n_kv_heads;
    return launch_copies(sources, positions, firsts, n_sources, destinations, k, v, slabs, slabs, 16, stream);
}

// data [entry][slot] of `bytes` bytes each, slots `slot_stride` bytes apart, entries `entry_stride`; lists as above, without positions.
extern "C" int b200_copy_slots(void* data, long long entry_stride, long long slot_stride, long long bytes, int n_entries, const int* sources,
                               const int* firsts, int n_sources, const int* destinations, cudaStream_t stream) {
    using namespace b200;
    if (n_sources <= 0 || n_entries <= 0 || bytes <= 0) return 0;
    const unsigned long long all = (unsigned long long)(uintptr_t)data | entry_stride | slot_stride | bytes;
    int width = 16;
    while (all % width) width /= 2;
    const long long per_index = (bytes + kStateSlab - 1) / kStateSlab;
    if (per_index * n_entries > 0x7fffffffll) return kErrUnsupportedSize;
    const Slabs s{(unsigned char*)data, entry_stride, slot_stride, kStateSlab, kStateSlab, bytes, (int)per_index, 1, kStateSlab};
    return launch_copies(sources, nullptr, firsts, n_sources, destinations, s, s, (int)per_index * n_entries, 0, width, stream);
}
