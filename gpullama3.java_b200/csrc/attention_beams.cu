// One decode step's attention of sequences that come in groups (the beams of a request) and share their first pages.
//
//   o[r, h] = softmax_j(q[r, h] . k[j, h / rep] / sqrt(D)) v[j, h / rep],   j < kv_len[r]  (with a window: j >= kv_len[r] - window)
//
// Groups are `beams` consecutive sequences; the first shared_pages[g] entries of their page-table rows name the same pages, all of
// them full.  Those are read once for all beams of the group and all query heads of a kv head, which are the rows of one
// tile: at 8 beams of 32 heads on 8 that is 32 rows, and an eighth of the bytes that as many separate sequences read.
//
// The work is cut by pages.  The pages of one segment belong together: the shared pages of a group, then the pages that each
// of its sequences has for itself, group after group.  All segments in this order make one line, on which a page is 1 long (in float32, where the tensor
// cores bound it, a shared one 2 or 4 with more than 16 or 32 rows) and a segment with pages kSegmentCost longer (what it costs to begin and leave one); of every kv head each of gridDim.x CTAs takes the pages of an equal
// stretch, whatever they belong to, so groups of unequal length share the GPU evenly.  The line is laid out by each CTA for itself, or once for all
// layers of a step by attention_beams_plan.
// A CTA keeps the running maximum m, sum l and output o of a segment's rows in registers and leaves them, unnormalised, in
// scratch at the segment's end or its own; a second kernel joins what the CTAs left of a row, in a fixed order.  CTA c's piece of
// segment s is number c + s (along the pages either grows, so no two pieces have one number).
//
// Fused variant (b200_attention_beams_rope): the step's own rotation and cache write are done here, as in the decode kernel for separate
// sequences: the queries are turned on their way into shared memory, and the CTA that meets a sequence's last page turns the new key, puts it and the new
// value into the page as it lies in shared memory and into the cache.  The page that holds the new position is always a sequence's own.
//
// Groups of more than 64 rows to a kv head are cut into equal groups of whole beams, each of which reads the shared pages.
//
// Bound by HBM in bytes: every key and value that some row reads, once.  Measured (both kernels, no plan given): 4 groups of 4 beams, 32 heads
// on 8 of 128, at 2,200 to 16,200 positions, 155 MB in 35.5 us, 5.4 TB/s while the pages stream; 8 groups of 8 beams, 32 heads on 8 of 64, at about
// 4,100 positions, 76 MB in 29.5 us: 2 us for the line, 1.5 until the first page is there, 20 of pages, 4.5 for the join and the rest for starts
// and ends; one group of 4 at 920 positions 8.6 us, of which the pages need 0.3.  float32 is bound by the tensor cores (six products for one, 57% of
// their rate while pages stream): 8 groups of 8 beams, 32 heads on 8 of 64, at about 3,900 positions, 144 MB in 72 us (178 us on
// multiply-adds, bound by reading queries and probabilities from shared memory).
#include "common.cuh"

namespace b200 {

constexpr int kBaThreads = 128;
constexpr int kBaRows = 64;             // most rows (beam, query head) of a tile
constexpr int kBaMaxSegments = 2048;
constexpr int kBaRing = 64, kBaKnown = 32;     // pages known ahead, so many looked up at a time

struct BeamAttnArgs {
    const void* q;
    void* out;
    const int* kv_lens;
    const int* page_table;
    const int* shared_pages;
    const void* k_pool;
    const void* v_pool;
    float* part_o;                      // [kv_head][piece][row][D]
    float* part_ml;                     // [kv_head][piece][row][2]
    int* plan;                          // the segments, as many ints as plan_ints
    int given;                          // whether they are there already
    const float* inv_freq;              // of the fused variant, [head_dim / 2], else null
    int pairing;                        // 0: (2j, 2j+1); 1: (j, j + head_dim/2)
    int write_cache;                    // whether the step's keys and values go into the cache here
    int fresh;                          // 1: the last position's key and value are not in the cache yet
    unsigned per_magic;                 // 2^32 / (sub_beams + 1), rounded up
    long long q_row_stride;
    int table_stride, n_seqs, n_groups, beams, sub_beams, n_sub, n_parts, n_segments, n_heads, n_kv_heads, window;
    int length;                         // of a shared page on the line of a plan that is made here, as a power of two
};

__device__ __forceinline__ int first_key(int kv_len, int window) { return window > 0 ? max(0, kv_len - window) : 0; }

// Segments: part p of n_parts = n_groups * n_sub (n_sub parts of up to sub_beams sequences to a group) has its shared pages as segment
// p * (sub_beams + 1), its sequences' own as the next ones.
__device__ __forceinline__ int part_first_row(const BeamAttnArgs& a, int p) {
    if (a.n_sub == 1) return p * a.beams;
    const int g = p / a.n_sub;
    return g * a.beams + (p - g * a.n_sub) * a.sub_beams;
}
__device__ __forceinline__ int part_rows(const BeamAttnArgs& a, int p) {
    return a.n_sub == 1 ? a.beams : min(a.sub_beams, a.beams - (p % a.n_sub) * a.sub_beams);
}

__device__ __forceinline__ int part_of_segment(const BeamAttnArgs& a, int s) { return (int)__umulhi((unsigned)s, a.per_magic); }   // (s below 2^16)

constexpr int kSegmentCost = 2;
struct Segment {
    int pages;          // pages before it
    int at;             // where it begins on the line
    int lo;             // its first page's place in the page table
    int row;            // the sequence whose row of the table that is
};
// In shared memory: [n_segments + 1] of these, the last one's `pages` and `at` the ends, its `row` the length of a shared page (2 to that power); then the sequences' lengths (as far as they are
// needed) and the parts' shared pages.
static int plan_ints(const BeamAttnArgs& a) { return 4 * (a.n_segments + 1) + a.n_seqs + 2 * a.n_parts; }
// the length of a segment's pages as a power of two, `shared` being that of the shared ones
__device__ __forceinline__ int page_length(const BeamAttnArgs& a, int s, int shared) {
    return shared == 0 || part_of_segment(a, s) * (a.sub_beams + 1) != s ? 0 : shared;
}
// the length of a CTA's stretch, `end` being the plan's last entry: no shorter than a page, so that every CTA between the first and the last one with
// pages of a segment has some
__device__ __forceinline__ int stretch_of(const Segment& end, int ctas) { return max(1 << end.row, (end.at + ctas - 1) / ctas); }

// Lays the line out.  By all threads of a CTA.  `tmp`: two ints for each warp.
template <int THREADS>
__device__ __forceinline__ void make_plan(const BeamAttnArgs& a, Segment* seg, int* lens, int* tmp) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* range = lens + a.n_seqs;
    for (int i = tid; i < a.n_seqs; i += THREADS) lens[i] = max(a.kv_lens[i], 0);
    for (int p = tid; p < a.n_parts; p += THREADS) range[2 * p + 1] = min(max(a.shared_pages[a.n_sub == 1 ? p : p / a.n_sub], 0), a.table_stride);
    __syncthreads();
    // shared pages: those that some sequence of the part reads, as far as they are full for all
    for (int p = tid; p < a.n_parts; p += THREADS) {
        const int r0 = part_first_row(a, p), n = part_rows(a, p);
        int shortest = lens[r0];
        for (int i = 1; i < n; ++i) shortest = min(shortest, lens[r0 + i]);
        const int hi = min(range[2 * p + 1], max(shortest - a.fresh, 0) / kPageTokens);
        range[2 * p] = min(first_key(shortest, a.window) / kPageTokens, hi);
        range[2 * p + 1] = hi;
    }
    __syncthreads();
    // a thread's consecutive segments: their pages are counted, then added up in order
    const int each = (a.n_segments + THREADS - 1) / THREADS, s0 = tid * each, s1 = min(a.n_segments, s0 + each);
    int pages = 0, line = 0;
    for (int s = s0; s < s1; ++s) {
        const int p = part_of_segment(a, s), i = s - p * (a.sub_beams + 1), r0 = part_first_row(a, p);
        int lo = range[2 * p], hi = range[2 * p + 1], row = r0;
        if (i > 0) {
            lo = hi;
            if (i <= part_rows(a, p)) {
                row = r0 + i - 1;
                const int len = lens[row];
                hi = min((len + kPageTokens - 1) / kPageTokens, a.table_stride);
                lo = min(max(lo, first_key(len, a.window) / kPageTokens), hi);
            }
        }
        seg[s] = Segment{hi - lo, 0, lo, row};
        pages += hi - lo;
        line += hi > lo ? ((hi - lo) << page_length(a, s, a.length)) + kSegmentCost : 0;
    }
    int pages_to = pages, line_to = line;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, pages_to, o), w = __shfl_up_sync(0xffffffffu, line_to, o);
        if (lane >= o) { pages_to += v; line_to += w; }
    }
    if (lane == 31) { tmp[2 * warp] = pages_to; tmp[2 * warp + 1] = line_to; }
    __syncthreads();
    int pages_before = pages_to - pages, line_before = line_to - line;
    for (int w = 0; w < warp; ++w) { pages_before += tmp[2 * w]; line_before += tmp[2 * w + 1]; }
    for (int s = s0; s < s1; ++s) {
        const int n = seg[s].pages;
        seg[s].pages = pages_before;
        seg[s].at = line_before;
        pages_before += n;
        line_before += n > 0 ? (n << page_length(a, s, a.length)) + kSegmentCost : 0;
    }
    if (tid == THREADS - 1) seg[a.n_segments] = Segment{pages_before, line_before, 0, a.length};
    __syncthreads();
}

// The same for a CTA that is given the plan, and for one that is not (CTA 0, 0 of those leaves it for the kernel that joins the pieces).
template <int THREADS>
__device__ __forceinline__ void take_plan(const BeamAttnArgs& a, Segment* seg, int* lens, int* tmp) {
    if (a.given) {
        for (int i = threadIdx.x; i <= a.n_segments; i += THREADS) reinterpret_cast<int4*>(seg)[i] = reinterpret_cast<const int4*>(a.plan)[i];
        for (int i = threadIdx.x; i < a.n_seqs; i += THREADS) lens[i] = max(a.kv_lens[i], 0);
        __syncthreads();
        return;
    }
    make_plan<THREADS>(a, seg, lens, tmp);
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i <= a.n_segments; i += THREADS) reinterpret_cast<int4*>(a.plan)[i] = reinterpret_cast<const int4*>(seg)[i];
}

__global__ void __launch_bounds__(256) attention_beams_plan_kernel(const __grid_constant__ BeamAttnArgs a) {
    extern __shared__ __align__(16) int plan_smem[];
    __shared__ int tmp[16];
    Segment* seg = reinterpret_cast<Segment*>(plan_smem);
    pdl_launch_dependents();
    pdl_wait();
    make_plan<256>(a, seg, plan_smem + 4 * (a.n_segments + 1), tmp);
    for (int i = threadIdx.x; i <= a.n_segments; i += 256) reinterpret_cast<int4*>(a.plan)[i] = reinterpret_cast<const int4*>(seg)[i];
}

// the segment of page number u: the last one that begins at or before it, which is not an empty one
__device__ __forceinline__ int segment_of(const BeamAttnArgs& a, const Segment* seg, int u) {
    int lo = 0, hi = a.n_segments - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seg[mid].pages <= u) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// the numbers of the pages that begin before places x and y of the line
__device__ __forceinline__ int2 pages_before(const BeamAttnArgs& a, const Segment* seg, int x, int y) {
    int lx = 0, hx = a.n_segments - 1, ly = 0, hy = hx;
    while (lx < hx || ly < hy) {
        const int mx = (lx + hx + 1) >> 1, my = (ly + hy + 1) >> 1;
        const int ax = seg[mx].at, ay = seg[my].at;
        if (lx < hx) { if (ax <= x) lx = mx; else hx = mx - 1; }
        if (ly < hy) { if (ay <= y) ly = my; else hy = my - 1; }
    }
    const int length = seg[a.n_segments].row;
    auto before = [&](int s, int z) {
        const int power = page_length(a, s, length);
        return seg[s].pages + min((max(z - seg[s].at - kSegmentCost, 0) + (1 << power) - 1) >> power, seg[s + 1].pages - seg[s].pages);
    };
    return make_int2(before(lx, x), before(ly, y));
}

// A page of the work: where it lies, whose it is, its first position, and how many of its keys there are.
struct Unit {
    int page, segment, position, keys;
};
__device__ __forceinline__ Unit unit_of(const BeamAttnArgs& a, const Segment* seg, const int* lens, int u) {
    Unit x;
    x.segment = segment_of(a, seg, u);
    const Segment s = seg[x.segment];
    const int index = s.lo + u - s.pages;
    x.page = a.page_table[(size_t)s.row * a.table_stride + index];
    x.position = index * kPageTokens;
    x.keys = min(kPageTokens, lens[s.row] - x.position);
    return x;
}

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, int bytes) {      // the rest of the 16 is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same without what was in d
__device__ __forceinline__ void mma_bf16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Both types on mma.sync.  A warp owns a tile of 16 rows and, where there are fewer than four tiles, a part of each page's keys.  Rows of shared memory
// are such that what lanes read together meets no bank twice: bfloat16, eight rows of an ldmatrix block in rows of 128 or 256 bytes with
// their 16-byte pieces exchanged by the row's last three bits, others with 16 bytes between them; float32, the halves of 128 bytes exchanged in
// every other row, of which two are read at a time.
template <typename E, int D>
struct BeamTile;
template <int D>
struct BeamTile<__nv_bfloat16, D> {
    static constexpr bool kExchange = D % 64 == 0;
    static constexpr int kPitchK = kExchange ? 2 * D : 2 * D + 16, kPitchV = 2 * kPageTokens, kPitchQ = kPitchK;       // bytes
    static constexpr int kStage = kPageTokens * kPitchK + D * kPitchV, kPeriod = 8;
    // As many stages as leave room for three CTAs an SM with heads of up to 64, two with wider ones.
    static constexpr int kResident = D <= 64 ? 3 : 2, kMore = D <= 64 ? 4 : 3;
    static __device__ __forceinline__ uint32_t k_piece(int row, int c) { return row * kPitchK + ((kExchange ? c ^ (row & 7) : c) << 4); }
    static __device__ __forceinline__ uint32_t v_piece(int row, int c) { return row * kPitchV + ((c ^ (row & 7)) << 4); }
};
template <int D>
struct BeamTile<float, D> {
    static constexpr int kPitchK = 4 * D, kPitchV = 4 * kPageTokens, kPlaneQ = 2 * D + 16, kPitchQ = 3 * kPlaneQ;       // (queries: three parts, see below)
    static constexpr int kStage = kPageTokens * kPitchK + D * kPitchV, kPeriod = 2;
    static constexpr int kResident = D <= 64 ? 2 : 1, kMore = 3;
    static __device__ __forceinline__ uint32_t k_piece(int row, int c) { return row * kPitchK + ((c ^ ((row & 1) << 2)) << 4); }
    static __device__ __forceinline__ uint32_t v_piece(int row, int c) { return row * kPitchV + ((c ^ ((row & 1) << 2)) << 4); }
};

template <int D>
struct RowState {
    float o[D / 8][4];
    float m[2], l[4];               // of rows g and g + 8; l twice each (float32: a lane's share in the first)
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
        m[0] = m[1] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = 0.f;
    }
};

// NK keys of a page, from its key `first` on, for the tile whose query fragments are qa.  Nothing is rescaled unless some row's maximum has grown.
template <int D, int NK>
__device__ __forceinline__ void attend_keys(RowState<D>& st, const uint32_t (&qa)[D / 16][4], uint32_t k_base, uint32_t v_base, int first, int lane,
                                            float scale_log2, bool masked, int position, const int (&row_lo)[2], int row_end) {
    constexpr int NT = NK / 8;
    using T = BeamTile<__nv_bfloat16, D>;
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][c] = 0.f;
    // ldmatrix: lanes 0-7, 8-15, 16-23, 24-31 give the rows of the four 8 x 8 blocks (keys 0-7 and 8-15 by 8 dimensions and the next 8)
    const int low = lane & 7, half = (lane >> 3) & 1, row = low + (lane >> 4) * 8;
    const uint32_t k_row = k_base + (uint32_t)((first + row) * T::kPitchK);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const int c = ks * 2 + half;
        const uint32_t piece = (uint32_t)((T::kExchange ? c ^ low : c) << 4);
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
            uint32_t kb[4];
            ldmatrix4(kb, k_row + piece + (uint32_t)(i * 8 * T::kPitchK));
            mma_bf16(s[i], qa[ks], kb[0], kb[1]);
            mma_bf16(s[i + 1], qa[ks], kb[2], kb[3]);
        }
    }
    if (masked) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = position + first + 8 * i + 2 * (lane & 3) + (c & 1);
                if (key < row_lo[c >> 1] || key >= row_end) s[i][c] = -INFINITY;
            }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c >> 1] = fmaxf(top[c >> 1], s[i][c]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2)) * scale_log2;
    }
    if (__any_sync(0xffffffffu, top[0] > st.m[0] || top[1] > st.m[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float m = fmaxf(st.m[h], top[h]), keep = m == -INFINITY ? 1.f : exp2_fast(st.m[h] - m);
            st.m[h] = m;
            st.l[2 * h] *= keep;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) { st.o[j][2 * h] *= keep; st.o[j][2 * h + 1] *= keep; }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float base = st.m[h] == -INFINITY ? 0.f : st.m[h];        // (a row that has seen nothing yet: its probabilities are 0)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[i][2 * h + e] = exp2_fast(fmaf(s[i][2 * h + e], scale_log2, -base));
    }
    const uint32_t v_row = v_base + (uint32_t)(row * T::kPitchV);
#pragma unroll
    for (int kk = 0; kk < NK / 16; ++kk) {
        // A probability goes to the tensor cores as two bfloat16 numbers, what it rounds to and what that leaves, 16 bits together; their sum, a product with
        // ones in 32 bits, is what it is divided by.  (In one number of 8 bits results are off by 1.7e-3 to 1.8e-3 of their norm against 64 bits, as
        // they are by 1.65e-3, their own rounding, and 8 groups of 8 beams at 4,100 positions take 26.1 us in place of 29.5, a step of theirs 1.42 ms
        // in place of 1.47.)
        const uint32_t pa[4] = {pack2(s[2 * kk][0], s[2 * kk][1]), pack2(s[2 * kk][2], s[2 * kk][3]),
                                pack2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        auto left = [&](uint32_t h, float x, float y) { return pack2(x - __uint_as_float(h << 16), y - __uint_as_float(h & 0xffff0000u)); };
        const uint32_t pr[4] = {left(pa[0], s[2 * kk][0], s[2 * kk][1]), left(pa[1], s[2 * kk][2], s[2 * kk][3]),
                                left(pa[2], s[2 * kk + 1][0], s[2 * kk + 1][1]), left(pa[3], s[2 * kk + 1][2], s[2 * kk + 1][3])};
        mma_bf16(st.l, pr, 0x3f803f80u, 0x3f803f80u);
        mma_bf16(st.l, pa, 0x3f803f80u, 0x3f803f80u);
        const uint32_t piece = (uint32_t)((((first >> 3) + kk * 2 + half) ^ low) << 4);
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
            uint32_t vb[4];
            ldmatrix4(vb, v_row + piece + (uint32_t)(j * 8 * T::kPitchV));
            mma_bf16(st.o[j], pr, vb[0], vb[1]);
            mma_bf16(st.o[j + 1], pr, vb[2], vb[3]);
            mma_bf16(st.o[j], pa, vb[0], vb[1]);
            mma_bf16(st.o[j + 1], pa, vb[2], vb[3]);
        }
    }
}

// float32: x = h + m + l, three bfloat16 numbers of 8 bits each (what is left is below 2^-26 of x); a product is h h + (h m + m h) + (m m + h l + l h),
// six on the tensor cores with an error below that of one product's rounding.  The three magnitudes are added separately, and the output of 16
// keys before it joins the row's, in 32 bits: a tensor core's own sum drops bits instead of rounding them.  Numbers from 2^-109 on have all three
// parts, smaller ones are held to 2^-134 (half of bfloat16's last place there).  What is not finite, or rounds to infinity in bfloat16 (from 3.39e38 on), gives
// NaN wherever it is multiplied, and the rows concerned are computed once more, on multiply-adds, where the pieces are joined.
struct Parts {
    uint32_t h, m, l;
};
__device__ __forceinline__ Parts parts_of(float x, float y) {
    Parts p;
    p.h = pack2(x, y);
    x -= __uint_as_float(p.h << 16);
    y -= __uint_as_float(p.h & 0xffff0000u);
    p.m = pack2(x, y);
    x -= __uint_as_float(p.m << 16);
    y -= __uint_as_float(p.m & 0xffff0000u);
    p.l = pack2(x, y);
    return p;
}
struct Sums {
    float s[3][4];
    // a: the parts of 16 rows by 16, [part][register]; b0, b1: the parts of two numbers each of this lane's column.  first: nothing has been added yet.
    __device__ __forceinline__ void add(bool first, const uint32_t (&a)[3][4], const Parts& b0, const Parts& b1) {
        if (first) {
            mma_bf16_zero(s[2], a[1], b0.m, b1.m);
            mma_bf16_zero(s[1], a[0], b0.m, b1.m);
            mma_bf16_zero(s[0], a[0], b0.h, b1.h);
        } else {
            mma_bf16(s[2], a[1], b0.m, b1.m);
            mma_bf16(s[1], a[0], b0.m, b1.m);
            mma_bf16(s[0], a[0], b0.h, b1.h);
        }
        mma_bf16(s[2], a[0], b0.l, b1.l);
        mma_bf16(s[1], a[1], b0.h, b1.h);
        mma_bf16(s[2], a[2], b0.h, b1.h);
    }
    __device__ __forceinline__ float total(int c) const { return s[0][c] + (s[1][c] + s[2][c]); }
};

// 16 keys of a page from its key `first` on.  Dimensions and keys are paired with the matrix instructions' places so that a lane's four numbers of a
// row are one access: place 2 t + e of sixteen is number 4 t + e, place 8 + 2 t + e number 4 t + 2 + e.  q_row: the lane's row of queries.
template <int D>
__device__ __forceinline__ void attend_keys_f32(RowState<D>& st, uint32_t q_row, const unsigned char* k_page, const unsigned char* v_page, int first, int lane,
                                                float scale, bool masked, int position, const int (&row_lo)[2], int row_end) {
    using T = BeamTile<float, D>;
    const int n = lane >> 2, t = lane & 3;
    Sums sums[2];
    const int key0 = first + 4 * (n >> 1) + (n & 1);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t qa[3][4];
#pragma unroll
        for (int p = 0; p < 3; ++p) ldmatrix4(qa[p], q_row + p * T::kPlaneQ + (ks * 2 + (lane >> 4)) * 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 k = *reinterpret_cast<const float4*>(k_page + T::k_piece(key0 + 2 * i, ks * 4 + t));
            sums[i].add(ks == 0, qa, parts_of(k.x, k.y), parts_of(k.z, k.w));
        }
    }
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            s[i][c] = sums[i].total(c) * scale;
            const int key = position + first + 4 * t + 2 * i + (c & 1);
            if (masked && (key < row_lo[c >> 1] || key >= row_end)) s[i][c] = -INFINITY;
        }
    float keep[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m = fmaxf(st.m[h], top), base = m == -INFINITY ? 0.f : m;       // (a row that has seen nothing yet: its probabilities are 0)
        keep[h] = expf(st.m[h] - base);
        st.m[h] = m;
        st.l[2 * h] *= keep[h];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[i][2 * h + e] = expf(s[i][2 * h + e] - base);
                st.l[2 * h] += s[i][2 * h + e];
            }
    }
    const Parts p0 = parts_of(s[0][0], s[0][1]), p1 = parts_of(s[0][2], s[0][3]), p2 = parts_of(s[1][0], s[1][1]), p3 = parts_of(s[1][2], s[1][3]);
    const uint32_t pa[3][4] = {{p0.h, p1.h, p2.h, p3.h}, {p0.m, p1.m, p2.m, p3.m}, {p0.l, p1.l, p2.l, p3.l}};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
        const float4 v = *reinterpret_cast<const float4*>(v_page + T::v_piece(8 * j + n, (first >> 2) + t));
        Sums o;
        o.add(true, pa, parts_of(v.x, v.y), parts_of(v.z, v.w));
#pragma unroll
        for (int c = 0; c < 4; ++c) st.o[j][c] = st.o[j][c] * keep[c >> 1] + o.total(c);
    }
}

// What a difference of maxima comes to: they are in units of log 2 where the scores were, in bfloat16.
template <typename E> __device__ __forceinline__ float weight(float x) { return sizeof(E) == 2 ? exp2_fast(x) : expf(x); }

// Joins the parts that the warps of a tile hold and stores the tile's first `rows` rows at `to_o` and `to_ml`.  All warps of the CTA call it.
template <typename E, int D>
__device__ __forceinline__ void leave_tile(RowState<D>& st, float* join, int parts, int part, int tile, int lane, int rows, float* to_o, float* to_ml) {
    constexpr int P = D + 4;
    const int g = lane >> 2, t = lane & 3;
    for (int half = parts / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (part >= half && part < 2 * half) {
            // (four parts: two of one tile; two parts: one each of two tiles)
            float* to = join + (parts == 2 ? tile : part - half) * 16 * P;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* row = to + (g + 8 * h) * P;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(row + 8 * j + 2 * t) = make_float2(st.o[j][2 * h], st.o[j][2 * h + 1]);
                if (t == 0) { row[D] = st.m[h]; row[D + 1] = st.l[2 * h]; }
            }
        }
        __syncthreads();
        if (part < half) {
            const float* from = join + (parts == 2 ? tile : part) * 16 * P;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float* row = from + (g + 8 * h) * P;
                const float m2 = row[D], l2 = row[D + 1], m = fmaxf(st.m[h], m2), base = m == -INFINITY ? 0.f : m;
                const float c1 = weight<E>(st.m[h] - base), c2 = weight<E>(m2 - base);
                st.m[h] = m;
                st.l[2 * h] = st.l[2 * h] * c1 + l2 * c2;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    const float2 o2 = *reinterpret_cast<const float2*>(row + 8 * j + 2 * t);
                    st.o[j][2 * h] = st.o[j][2 * h] * c1 + o2.x * c2;
                    st.o[j][2 * h + 1] = st.o[j][2 * h + 1] * c1 + o2.y * c2;
                }
            }
        }
    }
    if (part != 0) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = tile * 16 + g + 8 * h;
        if (r >= rows) continue;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(to_o + (size_t)r * D + 8 * j + 2 * t) = make_float2(st.o[j][2 * h], st.o[j][2 * h + 1]);
        if (t == 0) *reinterpret_cast<float2*>(to_ml + 2 * r) = make_float2(st.m[h], st.l[2 * h]);
    }
}

// STAGES pages are in shared memory or on their way there.  A piece's parts are joined in the stage that was read last.
// (The compiler is told how many CTAs share an SM but for wide bfloat16 heads, where it then takes 248 registers in place of 182 and the 4 groups of
// 4 beams above 37.6 us in place of 35.8.)
template <typename E, int D, int STAGES>
__global__ void __launch_bounds__(kBaThreads, sizeof(E) == 4 || D <= 64 ? BeamTile<E, D>::kResident : 0) attention_beams_kernel(const __grid_constant__ BeamAttnArgs a) {
    using T = BeamTile<E, D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int tmp[kBaThreads / 16];
    __shared__ Unit ring[kBaRing];
    unsigned char* q_s = smem + STAGES * T::kStage;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, rep = a.n_heads / a.n_kv_heads;
    float* turn_s = reinterpret_cast<float*>(q_s + a.sub_beams * rep * T::kPitchQ);     // fused: [sequence of the part][cosines, sines of its D / 2 angles]
    Segment* seg = reinterpret_cast<Segment*>(turn_s + (a.inv_freq ? a.sub_beams * D : 0));
    int* lens = reinterpret_cast<int*>(seg + a.n_segments + 1);
    pdl_wait();
    // (only now: the kernel that joins the pieces may read a given plan as soon as it starts)
    pdl_launch_dependents();
    take_plan<kBaThreads>(a, seg, lens, tmp);
    const int per = stretch_of(seg[a.n_segments], gridDim.x);
    const int2 mine = pages_before(a, seg, blockIdx.x * per, (blockIdx.x + 1) * per);
    const int u0 = mine.x, u1 = mine.y;
    if (u0 >= u1) return;

    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem), q_base = (uint32_t)__cvta_generic_to_shared(q_s);
    constexpr bool kWide = sizeof(E) == 4;
    constexpr int kEach = 16 / sizeof(E), CK = D / kEach, CV = kPageTokens / kEach;        // elements of 16 bytes, such pieces of a row
    auto know = [&](int u) {        // pages u .. u + 31 into the ring
        if (tid < kBaKnown && u + tid < u1) ring[(u + tid - u0) % kBaRing] = unit_of(a, seg, lens, u + tid);
    };
    auto issue = [&](int u) {
        if (u < u1) {
            const Unit x = ring[(u - u0) % kBaRing];
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % STAGES) * T::kStage), vs = ks + kPageTokens * T::kPitchK;
            const E* k = (const E*)a.k_pool + (size_t)x.page * page_elements + head_off;
            const E* v = (const E*)a.v_pool + (size_t)x.page * page_elements + head_off;
            constexpr int RK = kBaThreads / CK, RV = kBaThreads / CV;
            if (x.keys == kPageTokens && kBaThreads % CK == 0 && RK % T::kPeriod == 0) {   // a thread's pieces lie whole rows apart, at one place in them
                const uint32_t kt = ks + T::k_piece(tid / CK, tid % CK), vt = vs + T::v_piece(tid / CV, tid % CV);
                k += tid * kEach;
                v += tid * kEach;
#pragma unroll
                for (int i = 0; i < kPageTokens / RK; ++i) cp_async16(kt + i * RK * T::kPitchK, k + i * kBaThreads * kEach);
#pragma unroll
                for (int i = 0; i < D / RV; ++i) cp_async16(vt + i * RV * T::kPitchV, v + i * kBaThreads * kEach);
            } else {
                for (int i = tid; i < kPageTokens * CK; i += kBaThreads)
                    cp_async16(ks + T::k_piece(i / CK, i % CK), k + (size_t)i * kEach, i / CK < x.keys ? 16 : 0);
                // (values of positions past the sequence's end are read as zeros: a probability of 0 times what is not finite is not 0)
                for (int i = tid; i < D * CV; i += kBaThreads)
                    cp_async16(vs + T::v_piece(i / CV, i % CV), v + (size_t)i * kEach, min(16, max(0, (int)sizeof(E) * (x.keys - kEach * (i % CV)))));
            }
        }
        cp_async_commit();
    };
    auto turned = [&](const float* turn, float x0, float x1, int j, float& y0, float& y1) {
        const float cs = turn[j], sn = turn[D / 2 + j];
        y0 = __fmaf_rn(x0, cs, -__fmul_rn(x1, sn));     // (the second product is rounded: queries and keys alike, wherever they are turned)
        y1 = __fmaf_rn(x0, sn, __fmul_rn(x1, cs));
    };
    auto ask_queries = [&](int p) {     // of all rows of part p
        const int r0 = part_first_row(a, p);
        if constexpr (kWide) {
            const int n = part_rows(a, p) * rep * CK;
            for (int c0 = tid; c0 < n; c0 += 4 * kBaThreads) {          // (four asked for at once)
                float4 x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int c = min(c0 + k * kBaThreads, n - 1), row = c / CK, at = c % CK;
                    x[k] = *reinterpret_cast<const float4*>((const E*)a.q + (size_t)(r0 + row / rep) * a.q_row_stride + (size_t)(kvh * rep + row % rep) * D + at * 4);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int c = c0 + k * kBaThreads, row = c / CK, at = c % CK;
                    if (c >= n) continue;
                    const Parts p0 = parts_of(x[k].x, x[k].y), p1 = parts_of(x[k].z, x[k].w);
                    uint32_t* to = reinterpret_cast<uint32_t*>(q_s + row * T::kPitchQ + (at / 4) * 32 + (at % 4) * 4);
                    to[0] = p0.h; to[T::kPlaneQ / 4] = p0.m; to[2 * T::kPlaneQ / 4] = p0.l;
                    to[4] = p1.h; to[T::kPlaneQ / 4 + 4] = p1.m; to[2 * T::kPlaneQ / 4 + 4] = p1.l;
                }
            }
            return;
        } else {
        if (a.inv_freq) {
            const int n = part_rows(a, p);
            for (int c = tid; c < n * (D / 2); c += kBaThreads) {
                const int b = c / (D / 2), j = c % (D / 2);
                sincosf((float)(lens[r0 + b] - 1) * a.inv_freq[j], &turn_s[b * D + D / 2 + j], &turn_s[b * D + j]);
            }
            __syncthreads();
            // two pieces of a row at a time: neighbours, or a half row apart
            for (int c = tid; c < n * rep * (CK / 2); c += kBaThreads) {
                const int row = c / (CK / 2), at = c % (CK / 2), first = a.pairing == 0 ? 2 * at : at, second = a.pairing == 0 ? 2 * at + 1 : at + CK / 2;
                const __nv_bfloat16* from = (const __nv_bfloat16*)a.q + (size_t)(r0 + row / rep) * a.q_row_stride + (size_t)(kvh * rep + row % rep) * D;
                const uint4 x = *reinterpret_cast<const uint4*>(from + first * 8), y = *reinterpret_cast<const uint4*>(from + second * 8);
                const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                float v[16];
#pragma unroll
                for (int k = 0; k < 8; ++k) { v[2 * k] = __uint_as_float(w[k] << 16); v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
                const float* turn = turn_s + row / rep * D;
                if (a.pairing == 0) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) turned(turn, v[2 * k], v[2 * k + 1], at * 8 + k, v[2 * k], v[2 * k + 1]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) turned(turn, v[k], v[8 + k], at * 8 + k, v[k], v[8 + k]);
                }
                *reinterpret_cast<uint4*>(q_s + T::k_piece(row, first)) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
                *reinterpret_cast<uint4*>(q_s + T::k_piece(row, second)) = make_uint4(pack2(v[8], v[9]), pack2(v[10], v[11]), pack2(v[12], v[13]), pack2(v[14], v[15]));
            }
            return;
        }
        for (int c = tid; c < part_rows(a, p) * rep * CK; c += kBaThreads) {
            const int row = c / CK, at = c % CK;
            cp_async16(q_base + T::k_piece(row, at), (const __nv_bfloat16*)a.q + (size_t)(r0 + row / rep) * a.q_row_stride
                                                         + (size_t)(kvh * rep + row % rep) * D + at * 8);
        }
        }
    };
    know(u0);
    __syncthreads();
    int part_of = part_of_segment(a, ring[0].segment);
    const bool made = kWide || a.inv_freq;
    if (!made) ask_queries(part_of);                     // (they arrive with the first page)
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(u0 + i);
    if (made) ask_queries(part_of);                      // (made while the first pages are on their way)

    const float scale = kWide ? 1.f / sqrtf((float)D) : 1.4426950408889634f / sqrtf((float)D);
    RowState<D> st;
    uint32_t qa[kWide ? 1 : D / 16][4], q_row = 0;
    int segment = -1, parts = 1, part = 0, tile = warp, rows = 0, lo_max = 0, row_end = 0, row_lo[2] = {0, 0};
    auto leave = [&](int u) {           // behind page u - 1, with its stage to join in
        const size_t piece = (size_t)kvh * (gridDim.x + a.n_segments) + blockIdx.x + segment;
        if constexpr (kWide) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                st.l[2 * h] += __shfl_xor_sync(0xffffffffu, st.l[2 * h], 1);
                st.l[2 * h] += __shfl_xor_sync(0xffffffffu, st.l[2 * h], 2);
            }
        }
        leave_tile<E, D>(st, reinterpret_cast<float*>(smem + ((u - 1 - u0) % STAGES) * T::kStage), parts, part, tile, lane, rows,
                      a.part_o + piece * kBaRows * D, a.part_ml + piece * kBaRows * 2);
    };
    for (int u = u0; u < u1; ++u) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        const Unit x = ring[(u - u0) % kBaRing];
        if (x.segment != segment) {
            if (segment >= 0) {
                leave(u);
                __syncthreads();
            }
            segment = x.segment;
            st.clear();
            const int p = part_of_segment(a, segment), i = segment - p * (a.sub_beams + 1), r0 = part_first_row(a, p), n = part_rows(a, p);
            if (p != part_of) {
                part_of = p;
                ask_queries(p);
                cp_async_commit();
                cp_async_wait<0>();
                __syncthreads();
            }
            rows = i == 0 ? n * rep : rep;
            parts = rows <= 16 ? 4 : rows <= 32 ? 2 : 1;
            tile = warp % (4 / parts);
            part = warp / (4 / parts);
            row_end = i == 0 ? 0x7fffffff : lens[r0 + i - 1];
            lo_max = 0;
            if (a.window > 0) {
                for (int b = 0; b < n; ++b) lo_max = max(lo_max, first_key(lens[r0 + b], a.window));
                if (i > 0) lo_max = first_key(row_end, a.window);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    row_lo[h] = i > 0 ? lo_max : first_key(lens[r0 + min(tile * 16 + (lane >> 2) + 8 * h, rows - 1) / rep], a.window);
            }
            // (rows behind the last one are its copies, and nothing of them is stored)
            const int row = min(tile * 16 + (lane & 15), rows - 1) + (i == 0 ? 0 : (i - 1) * rep);
            if constexpr (kWide) {
                q_row = q_base + row * T::kPitchQ;
            } else {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) ldmatrix4(qa[ks], q_base + T::k_piece(row, ks * 2 + (lane >> 4)));
            }
        }
        const int ahead = u + STAGES - 1;
        if (ahead < u1 && (ahead - u0) % kBaKnown == 0) {
            know(ahead);
            __syncthreads();
        }
        issue(ahead);
        if constexpr (!kWide) if (a.write_cache && row_end - x.position <= kPageTokens) {      // a sequence's last page: its new key and value
            const Segment own = seg[segment];
            const int slot = (u - u0) % STAGES, new_at = x.keys - 1, beam = own.row - part_first_row(a, part_of);
            const __nv_bfloat16* k_raw = (const __nv_bfloat16*)a.q + (size_t)own.row * a.q_row_stride + (size_t)(a.n_heads + kvh) * D;
            const __nv_bfloat16* v_raw = k_raw + (size_t)a.n_kv_heads * D;
            __nv_bfloat16* k = (__nv_bfloat16*)a.k_pool + (size_t)x.page * page_elements + head_off + (size_t)new_at * D;
            __nv_bfloat16* v = (__nv_bfloat16*)a.v_pool + (size_t)x.page * page_elements + head_off + new_at;
            unsigned char* ks = smem + slot * T::kStage;
            unsigned char* vs = ks + kPageTokens * T::kPitchK;
            for (int j = tid; j < D / 2; j += kBaThreads) {
                const int d[2] = {a.pairing == 0 ? 2 * j : j, a.pairing == 0 ? 2 * j + 1 : j + D / 2};
                float y[2];
                turned(turn_s + beam * D, __bfloat162float(k_raw[d[0]]), __bfloat162float(k_raw[d[1]]), j, y[0], y[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const __nv_bfloat16 key = __float2bfloat16_rn(y[e]), value = v_raw[d[e]];
                    k[d[e]] = key;
                    v[(size_t)d[e] * kPageTokens] = value;
                    *reinterpret_cast<__nv_bfloat16*>(ks + T::k_piece(new_at, d[e] / 8) + (d[e] % 8) * 2) = key;
                    *reinterpret_cast<__nv_bfloat16*>(vs + T::v_piece(d[e], new_at / 8) + (new_at % 8) * 2) = value;
                }
            }
            __syncthreads();
        }
        if (tile * 16 < rows) {
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % STAGES) * T::kStage), vs = ks + kPageTokens * T::kPitchK;
            const bool masked = x.keys < kPageTokens || x.position < lo_max;
            if constexpr (kWide) {
                const unsigned char* page = smem + ((u - u0) % STAGES) * T::kStage;
#pragma unroll 1
                for (int first = part * 16; first < kPageTokens; first += parts * 16)
                    attend_keys_f32<D>(st, q_row, page, page + kPageTokens * T::kPitchK, first, lane, scale, masked, x.position, row_lo, row_end);
            } else if (parts == 4) {
                attend_keys<D, 16>(st, qa, ks, vs, part * 16, lane, scale, masked, x.position, row_lo, row_end);
            } else {
#pragma unroll 1
                for (int first = part * 32; first < kPageTokens; first += parts * 32)
                    attend_keys<D, 32>(st, qa, ks, vs, first, lane, scale, masked, x.position, row_lo, row_end);
            }
        }
    }
    cp_async_wait<0>();
    leave(u1);
}

// One row from the keys that it sees and nothing else, in 32 bits: for rows that are not numbers, or have no weight, in what the tiles left.  There
// a number that is not finite (in float32, one that has no parts) comes to NaN in rows that do not see it too, as 0 times itself, and in rows that do, as
// it meets the parts of a probability one by one.
// By a warp, a lane a key of 32 at a time, then a lane D / 32 dimensions.  q_s: D floats of the warp's own.  (Slow: where all rows of 64 sequences of 3,900
// positions with 32 heads of 64 are such, 6.7 ms, 9.6 in float32.  A call without such rows takes as long as it did without this.)
template <typename T, int D>
__device__ __noinline__ void attend_row(const BeamAttnArgs& a, int seq, int head, float* q_s) {
    constexpr int E = D / 32, kEach = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, kvh = head / (a.n_heads / a.n_kv_heads);
    const int len = a.kv_lens[seq], end = min(len, a.table_stride * kPageTokens), lo = first_key(len, a.window);
    const T* q = (const T*)a.q + (size_t)seq * a.q_row_stride + (size_t)head * D;
    for (int d = lane; d < D; d += 32) {
        float x = to_f32<T>(q[d]);
        if (a.inv_freq) {               // (as in the tiles: see `turned`)
            const int j = a.pairing == 0 ? d / 2 : d % (D / 2);
            const bool second = a.pairing == 0 ? d % 2 != 0 : d >= D / 2;
            const float other = to_f32<T>(q[a.pairing == 0 ? d ^ 1 : (d + D / 2) % D]);
            float sn, cs;
            sincosf((float)(len - 1) * a.inv_freq[j], &sn, &cs);
            x = to_f32<T>(from_f32<T>(second ? __fmaf_rn(other, sn, __fmul_rn(x, cs)) : __fmaf_rn(x, cs, -__fmul_rn(other, sn))));
        }
        q_s[d] = x;
    }
    __syncwarp();
    const float scale = 1.f / sqrtf((float)D);
    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int k0 = lo / 32 * 32; k0 < end; k0 += 32) {
        const size_t page = (size_t)a.page_table[(size_t)seq * a.table_stride + k0 / kPageTokens] * page_elements + head_off;
        const int at = k0 % kPageTokens, key = k0 + lane;
        const bool seen = key >= lo && key < end;
        float s = -INFINITY;
        if (seen) {
            const uint4* k = reinterpret_cast<const uint4*>((const T*)a.k_pool + page + (size_t)(at + lane) * D);
            s = 0.f;
#pragma unroll 4
            for (int c = 0; c < D / kEach; ++c) {
                const uint4 w = k[c];
                const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
                for (int i = 0; i < kEach; ++i) s = fmaf(q_s[c * kEach + i], to_f32<T>(x[i]), s);
            }
            s *= scale;
        }
        const float top = fmaxf(m, warp_max(s)), base = top == -INFINITY ? 0.f : top;
        const float keep = expf(m - base), p = seen ? expf(s - base) : 0.f;
        m = top;
        l = l * keep + warp_sum(p);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= keep;
        const T* v = (const T*)a.v_pool + page + (size_t)lane * kPageTokens + at;
        for (int i = max(lo - k0, 0); i < min(32, end - k0); ++i) {
            const float w = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, to_f32<T>(v[(size_t)e * 32 * kPageTokens + i]), o[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) ((T*)a.out)[((size_t)seq * a.n_heads + head) * D + e * 32 + lane] = from_f32<T>(o[e] / l);
}

// A warp per (sequence, query head): the pieces that hold the row, first those of the shared pages, then of its own.  A lane reads a piece's maximum
// and sum; the outputs are asked for eight pieces at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_beams_join_kernel(const __grid_constant__ BeamAttnArgs a, int n_ctas) {
    constexpr int E = D / 32, kAtOnce = 8;
    __shared__ float q_s[4][D];         // (of rows that are computed once more)
    const int lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5), rep = a.n_heads / a.n_kv_heads;
    const int seq = at / a.n_heads, head = at - seq * a.n_heads, kvh = head / rep, in_group = head - kvh * rep;
    const int g = seq / a.beams, beam = seq - g * a.beams, sub = a.n_sub == 1 ? 0 : beam / a.sub_beams, i = beam - sub * a.sub_beams;
    const int shared = (g * a.n_sub + sub) * (a.sub_beams + 1), own = shared + 1 + i;
    const bool mine = at < a.n_seqs * a.n_heads;
    pdl_launch_dependents();
    if (!a.given) pdl_wait();       // (a given plan was complete before the kernel ahead of this one began its work)
    const Segment* seg = reinterpret_cast<const Segment*>(a.plan);
    int c0 = 0, n0 = 0, c1 = 0, n1 = 0;     // the first CTA with pages of the shared segment and their number; the same of its own
    if (mine) {
        const int2* of = reinterpret_cast<const int2*>(seg);        // (pages, at) of each
        const int2 s0 = of[2 * shared], s1 = of[2 * shared + 2], o0 = of[2 * own], o1 = of[2 * own + 2];
        const Segment end = seg[a.n_segments];
        const unsigned per = (unsigned)stretch_of(end, n_ctas), magic = per > 1 ? 0xffffffffu / per + 1u : 0u;
        auto cta_of = [&](int x) {              // x / per
            if (magic == 0u) return x;
            const unsigned q = __umulhi((unsigned)x, magic);
            return (int)((unsigned long long)q * per > (unsigned)x ? q - 1u : q);
        };
        const int sa = s0.y + kSegmentCost, oa = o0.y + kSegmentCost, sn = s1.x - s0.x, on = o1.x - o0.x;
        c0 = cta_of(sa);
        n0 = sn > 0 ? cta_of(sa + ((sn - 1) << end.row)) - c0 + 1 : 0;
        c1 = cta_of(oa);
        n1 = on > 0 ? cta_of(oa + on - 1) - c1 + 1 : 0;
    }
    if (a.given) pdl_wait();
    if (!mine) return;
    const int n = n0 + n1;
    const size_t base = (size_t)kvh * (n_ctas + a.n_segments);
    auto row_of = [&](int k) {          // of the row in its k-th piece
        return k < n0 ? (base + c0 + k + shared) * kBaRows + i * rep + in_group : (base + c1 + (k - n0) + own) * kBaRows + in_group;
    };
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int k0 = 0; k0 < n; k0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (k0 + lane < n) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * row_of(k0 + lane));
        const float top = fmaxf(m, warp_max(ml.x)), zero = top == -INFINITY ? 0.f : top, keep = weight<T>(m - zero), f = weight<T>(ml.x - zero);
        l = l * keep + warp_sum(ml.y * f);
        m = top;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= keep;
        for (int k1 = 0; k1 < min(32, n - k0); k1 += kAtOnce) {
            float v[kAtOnce][E];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float* from = a.part_o + row_of(min(k0 + k1 + k, n - 1)) * D + lane;
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] = from[e * 32];
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float w = __shfl_sync(0xffffffffu, f, k1 + k);      // (0 behind the last piece)
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += v[k][e] * w;
            }
        }
    }
    bool lost = n > 0 && !(l > 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) lost = lost || isnan(o[e]);
    if (__any_sync(0xffffffffu, lost)) {
        attend_row<T, D>(a, seq, head, q_s[threadIdx.x >> 5]);
        return;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;      // (a sequence without keys: zeros)
#pragma unroll
    for (int e = 0; e < E; ++e) ((T*)a.out)[(size_t)at * D + e * 32 + lane] = from_f32<T>(o[e] * inv);
}

// sequences of a part: all beams of a group, or equal shares of them with at most 64 rows
static int beams_of_part(int beams, int rep) {
    const int n_sub = (beams * rep + kBaRows - 1) / kBaRows;
    int sub = (beams + n_sub - 1) / n_sub;
    if (sub * rep > kBaRows) sub = kBaRows / rep;
    return sub;
}
static long long segments_of(int n_groups, int beams, int rep) {
    const int sub = beams_of_part(beams, rep);
    return (long long)n_groups * ((beams + sub - 1) / sub) * (sub + 1);
}
static long long scratch_floats_of(int n_groups, int beams, int n_heads, int n_kv_heads, int head_dim, int n_parts) {
    const long long segments = segments_of(n_groups, beams, n_heads / n_kv_heads);
    return (segments + n_parts) * n_kv_heads * kBaRows * (head_dim + 2) + 4 * (segments + 1);
}
static int fill_args(BeamAttnArgs& a, const int* kv_lens, const int* shared_pages, int table_stride, int n_groups, int beams, int n_heads, int n_kv_heads,
                     int window, int dtype) {
    if (beams < 1 || n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads != 0 || window < 0 || table_stride < 1) return kErrBadArgument;
    const int rep = n_heads / n_kv_heads;
    if (rep > 16 || n_kv_heads > 65535) return kErrUnsupportedSize;
    if (segments_of(n_groups, beams, rep) > kBaMaxSegments) return kErrUnsupportedSize;
    a = BeamAttnArgs{};
    a.kv_lens = kv_lens; a.shared_pages = shared_pages;
    a.table_stride = table_stride; a.n_seqs = n_groups * beams; a.n_groups = n_groups; a.beams = beams;
    a.sub_beams = beams_of_part(beams, rep);
    a.n_sub = (beams + a.sub_beams - 1) / a.sub_beams;
    a.n_parts = n_groups * a.n_sub; a.n_segments = (int)segments_of(n_groups, beams, rep);
    a.per_magic = (unsigned)(((1ull << 32) + a.sub_beams) / (a.sub_beams + 1));
    a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.window = window;
    a.length = dtype == kF32 ? (a.sub_beams * rep > 32 ? 2 : a.sub_beams * rep > 16 ? 1 : 0) : 0;
    return 0;
}

constexpr int kSmShared = 228 * 1024, kCtaShared = 227 * 1024, kCtaReserved = 1024;      // bytes of an SM, the most of a CTA's, what each takes besides
constexpr int kStaticShared = 16 + kBaRing * (int)sizeof(Unit) + 1024;                      // at most, of attention_beams_kernel

template <typename Kernel>
static int launch_beams(Kernel kernel, void (*join)(const BeamAttnArgs, int), int smem, bool (&configured)[64], const BeamAttnArgs& a, int n_ctas,
                        cudaStream_t stream) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kErrBadArgument;
    if (!configured[device]) {          // the most that any call takes: of two threads that set it at once neither takes it back
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCtaShared - kStaticShared);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        configured[device] = true;
    }
    const int st = launch_pdl(kernel, dim3(n_ctas, a.n_kv_heads), dim3(kBaThreads), smem, stream, a);
    if (st != 0) return st;
    const long long rows = (long long)a.n_seqs * a.n_heads;
    return launch_pdl(join, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, a, n_ctas);
}

// bytes of dynamic shared memory with that many stages
template <typename E, int D>
static int beam_smem(const BeamAttnArgs& a, int stages) {
    using T = BeamTile<E, D>;
    return stages * T::kStage + a.sub_beams * ((a.n_heads / a.n_kv_heads) * T::kPitchQ + (a.inv_freq ? D * 4 : 0)) + plan_ints(a) * 4;
}

template <typename E, int D>
static int launch_beams_of(const BeamAttnArgs& a, int n_ctas, cudaStream_t stream) {
    using T = BeamTile<E, D>;
    static bool configured[2][64] = {};
    const auto join = attention_beams_join_kernel<E, D>;
    const int smem = beam_smem<E, D>(a, T::kMore), fewer = beam_smem<E, D>(a, 2);
    if (smem + kStaticShared + kCtaReserved <= kSmShared / T::kResident)
        return launch_beams(attention_beams_kernel<E, D, T::kMore>, join, smem, configured[0], a, n_ctas, stream);
    if (fewer + kStaticShared > kCtaShared) return kErrUnsupportedSize;
    return launch_beams(attention_beams_kernel<E, D, 2>, join, fewer, configured[1], a, n_ctas, stream);
}
template <int D>
static int launch_beams_of(int dtype, const BeamAttnArgs& a, int n_ctas, cudaStream_t stream) {
    return dtype == kF32 ? launch_beams_of<float, D>(a, n_ctas, stream) : launch_beams_of<__nv_bfloat16, D>(a, n_ctas, stream);
}

}  // namespace b200

extern "C" long long b200_attention_beams_scratch_floats(int n_groups, int beams, int n_heads, int n_kv_heads, int head_dim, int n_parts) {
    if (n_groups < 1 || beams < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads / n_kv_heads > 16) return 0;
    return b200::scratch_floats_of(n_groups, beams, n_heads, n_kv_heads, head_dim, n_parts);
}

// Ints of a plan (see below) for so many sequences in groups.
extern "C" int b200_attention_beams_plan_ints(int n_groups, int beams, int n_heads, int n_kv_heads) {
    if (n_groups < 1 || beams < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads / n_kv_heads > 16) return 0;
    return (int)(4 * (b200::segments_of(n_groups, beams, n_heads / n_kv_heads) + 1));
}

// The plan alone, for the layers of a step that share lengths, shared pages, heads and window.  fresh: 1 for the fused variant that writes the
// cache (the page that holds the last position is then no shared one, whatever shared_pages says).
extern "C" int b200_attention_beams_plan(int* plan, const int* kv_lens, const int* shared_pages, int table_stride, int n_groups, int beams, int n_heads,
                                         int n_kv_heads, int window, int dtype, int fresh, cudaStream_t stream) {
    using namespace b200;
    if (n_groups <= 0) return 0;
    BeamAttnArgs a;
    const int st = fill_args(a, kv_lens, shared_pages, table_stride, n_groups, beams, n_heads, n_kv_heads, window, dtype);
    if (st != 0) return st;
    if (dtype != kF32 && dtype != kBF16) return kErrBadArgument;
    if (((uintptr_t)plan & 15) != 0) return kErrUnsupportedSize;
    a.plan = plan;
    a.fresh = fresh != 0;
    // (segments are parts and sequences together, and a part has a sequence at least: sequences and parts twice are at most half as many again)
    static_assert((4 * (kBaMaxSegments + 1) + 3 * kBaMaxSegments / 2) * 4 <= 48 * 1024, "a plan fits the shared memory that needs no asking");
    return launch_pdl(attention_beams_plan_kernel, dim3(1), dim3(256), plan_ints(a) * 4, stream, a);
}

namespace b200 {

static int attention_beams(const void* q, long long q_row_stride, void* out, const int* kv_lens, const int* page_table, int table_stride,
                           const int* shared_pages, const void* k_pool, const void* v_pool, float* scratch, long long scratch_floats, int n_groups, int beams,
                           int n_heads, int n_kv_heads, int head_dim, int window, int n_parts, int dtype, const int* plan, const float* inv_freq, int pairing,
                           int write_cache, cudaStream_t stream) {
    if (n_groups <= 0) return 0;
    BeamAttnArgs a;
    const int st = fill_args(a, kv_lens, shared_pages, table_stride, n_groups, beams, n_heads, n_kv_heads, window, dtype);
    if (st != 0) return st;
    if ((dtype != kF32 && dtype != kBF16) || n_parts < 1 || pairing < 0 || pairing > 1) return kErrBadArgument;
    if (head_dim % 32 != 0 || head_dim < 32 || head_dim > 128 || n_parts > 65535 || (long long)a.n_seqs * n_heads > (1 << 28)) return kErrUnsupportedSize;
    if (q_row_stride % (dtype == kBF16 ? 8 : 4) != 0 || (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch | (uintptr_t)plan) & 15) != 0)
        return kErrUnsupportedSize;
    if (scratch_floats < scratch_floats_of(n_groups, beams, n_heads, n_kv_heads, head_dim, n_parts)) return 10003;
    a.q = q; a.out = out; a.page_table = page_table; a.k_pool = k_pool; a.v_pool = v_pool;
    a.q_row_stride = q_row_stride;
    a.inv_freq = inv_freq; a.pairing = pairing; a.write_cache = inv_freq && write_cache; a.fresh = a.write_cache;
    const long long pieces = (long long)(a.n_segments + n_parts) * n_kv_heads;
    a.part_o = scratch;
    a.part_ml = scratch + pieces * kBaRows * head_dim;
    a.given = plan != nullptr;
    a.plan = plan ? const_cast<int*>(plan) : (int*)(a.part_ml + pieces * kBaRows * 2);
    switch (head_dim) {
        case 32: return launch_beams_of<32>(dtype, a, n_parts, stream);
        case 64: return launch_beams_of<64>(dtype, a, n_parts, stream);
        case 96: return launch_beams_of<96>(dtype, a, n_parts, stream);
        default: return launch_beams_of<128>(dtype, a, n_parts, stream);
    }
}

}  // namespace b200

// Sequences are n_groups groups of `beams`; kv_lens[n_seqs], page_table [n_seqs][table_stride], shared_pages[n_groups].  n_parts: CTAs of
// a kv head.  plan: null, or what b200_attention_beams_plan made of the same numbers.  Keys and values of the step are in the cache already.
extern "C" int b200_attention_beams(const void* q, long long q_row_stride, void* out, const int* kv_lens, const int* page_table, int table_stride,
                                    const int* shared_pages, const void* k_pool, const void* v_pool, float* scratch, long long scratch_floats,
                                    int n_groups, int beams, int n_heads, int n_kv_heads, int head_dim, int window, int n_parts,
                                    int dtype, const int* plan, cudaStream_t stream) {
    return b200::attention_beams(q, q_row_stride, out, kv_lens, page_table, table_stride, shared_pages, k_pool, v_pool, scratch, scratch_floats, n_groups,
                                 beams, n_heads, n_kv_heads, head_dim, window, n_parts, dtype, plan, nullptr, 0, 0, stream);
}

// The fused variant, bfloat16: `qkv` holds the step's raw projections [n_seqs, (n_heads + 2 n_kv_heads) head_dim]; queries are turned here, and with
// write_cache the new key (turned) and value are stored at position kv_len - 1.  Rotary dimension = head_dim.
extern "C" int b200_attention_beams_rope(const void* qkv, long long q_row_stride, void* out, const int* kv_lens, const int* page_table, int table_stride,
                                         const int* shared_pages, void* k_pool, void* v_pool, float* scratch, long long scratch_floats, int n_groups,
                                         int beams, int n_heads, int n_kv_heads, int head_dim, int window, int n_parts, const int* plan,
                                         const float* inv_freq, int pairing, int write_cache, cudaStream_t stream) {
    if (inv_freq == nullptr) return b200::kErrBadArgument;
    return b200::attention_beams(qkv, q_row_stride, out, kv_lens, page_table, table_stride, shared_pages, k_pool, v_pool, scratch, scratch_floats, n_groups,
                                 beams, n_heads, n_kv_heads, head_dim, window, n_parts, b200::kBF16, plan, inv_freq, pairing, write_cache, stream);
}
