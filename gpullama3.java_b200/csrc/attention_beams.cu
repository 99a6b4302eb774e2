// One decode step's attention of sequences that come in groups (the beams of a request) and share their first pages.
//
//   o[r, h] = softmax_j(q[r, h] . k[j, h / rep] / sqrt(D)) v[j, h / rep],   j < kv_len[r]  (with a window: j >= kv_len[r] - window)
//
// Groups are `beams` consecutive sequences; the first shared_pages[g] entries of their page-table rows name the same pages, all of
// them full.  Those are read once for all beams of the group and all query heads of a kv head, which are the rows of one
// tile: at 8 beams of 32 heads on 8 that is 32 rows, and an eighth of the bytes that as many separate sequences read.
//
// The work is cut by pages.  The pages of one segment belong together: the shared pages of a group, then the pages that each
// of its sequences has for itself, group after group.  All segments in this order make one line, on which a page is 1 long and a segment with
// pages kSegmentCost longer (what it costs to begin and leave one); of every kv head each of gridDim.x CTAs takes the pages of an equal
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
// In shared memory: [n_segments + 1] of these, the last one's `pages` and `at` the ends; then the sequences' lengths (as far as they are
// needed) and the parts' shared pages.
static int plan_ints(const BeamAttnArgs& a) { return 4 * (a.n_segments + 1) + a.n_seqs + 2 * a.n_parts; }
// the length of a CTA's stretch
__device__ __forceinline__ int stretch_of(int line, int ctas) { return max(1, (line + ctas - 1) / ctas); }

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
        line += hi > lo ? hi - lo + kSegmentCost : 0;
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
        line_before += n > 0 ? n + kSegmentCost : 0;
    }
    if (tid == THREADS - 1) seg[a.n_segments] = Segment{pages_before, line_before, 0, 0};
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
    auto before = [&](int s, int z) { return seg[s].pages + min(max(z - seg[s].at - kSegmentCost, 0), seg[s + 1].pages - seg[s].pages); };
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
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// bfloat16, on mma.sync.  A warp owns a tile of 16 rows and, where there are fewer than four tiles, a part of each page's keys.  Rows of shared
// memory are such that the eight rows of an ldmatrix block meet no bank twice: 128 or 256 bytes with their 16-byte pieces exchanged
// by the row's last three bits, others with 16 bytes between them.
template <int D>
struct BeamTile {
    static constexpr bool kExchange = D % 64 == 0;
    static constexpr int kPitchK = kExchange ? 2 * D : 2 * D + 16, kPitchV = 2 * kPageTokens;       // bytes
    static constexpr int kStage = kPageTokens * kPitchK + D * kPitchV;
    static __device__ __forceinline__ uint32_t k_piece(int row, int c) { return row * kPitchK + ((kExchange ? c ^ (row & 7) : c) << 4); }
    static __device__ __forceinline__ uint32_t v_piece(int row, int c) { return row * kPitchV + ((c ^ (row & 7)) << 4); }
};

template <int D>
struct RowState {
    float o[D / 8][4];
    float m[2], l[4];               // of rows g and g + 8; l twice each
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

// NK keys of a page, from its key `first` on, for the tile whose query fragments are qa.  Nothing is rescaled unless some row's maximum has grown.  (To
// let it grow by 2^8 before it is followed saves 0.7 us of 28, and costs bits: a row's largest weight is then rounded like any other, where it
// is exactly 1 otherwise; against 64 bits 2.2e-3 of the norm in place of 1.8e-3, the rounding of the results alone being 1.7e-3.)
template <int D, int NK>
__device__ __forceinline__ void attend_keys(RowState<D>& st, const uint32_t (&qa)[D / 16][4], uint32_t k_base, uint32_t v_base, int first, int lane,
                                            float scale_log2, bool masked, int position, const int (&row_lo)[2], int row_end) {
    constexpr int NT = NK / 8;
    using T = BeamTile<D>;
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
        // Probabilities are rounded to bfloat16 for the tensor cores, as the values are stored.  Their sum is that of the rounded ones (in 32 bits,
        // a product with ones): what rounding adds to the weight of a key, it then adds to the sum as well.
        const uint32_t pa[4] = {pack2(s[2 * kk][0], s[2 * kk][1]), pack2(s[2 * kk][2], s[2 * kk][3]),
                                pack2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        mma_bf16(st.l, pa, 0x3f803f80u, 0x3f803f80u);
        const uint32_t piece = (uint32_t)((((first >> 3) + kk * 2 + half) ^ low) << 4);
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
            uint32_t vb[4];
            ldmatrix4(vb, v_row + piece + (uint32_t)(j * 8 * T::kPitchV));
            mma_bf16(st.o[j], pa, vb[0], vb[1]);
            mma_bf16(st.o[j + 1], pa, vb[2], vb[3]);
        }
    }
}

// Joins the parts that the warps of a tile hold and stores the tile's first `rows` rows at `to_o` and `to_ml`.  All warps of the CTA call it.
template <int D>
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
                const float c1 = exp2_fast(st.m[h] - base), c2 = exp2_fast(m2 - base);
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
template <int D, int STAGES>
__global__ void __launch_bounds__(kBaThreads) attention_beams_kernel(const __grid_constant__ BeamAttnArgs a) {
    using T = BeamTile<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int tmp[kBaThreads / 16];
    __shared__ Unit ring[kBaRing];
    unsigned char* q_s = smem + STAGES * T::kStage;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, rep = a.n_heads / a.n_kv_heads;
    float* turn_s = reinterpret_cast<float*>(q_s + a.sub_beams * rep * T::kPitchK);     // fused: [sequence of the part][cosines, sines of its D / 2 angles]
    Segment* seg = reinterpret_cast<Segment*>(turn_s + (a.inv_freq ? a.sub_beams * D : 0));
    int* lens = reinterpret_cast<int*>(seg + a.n_segments + 1);
    pdl_wait();
    // (only now: the kernel that joins the pieces may read a given plan as soon as it starts)
    pdl_launch_dependents();
    take_plan<kBaThreads>(a, seg, lens, tmp);
    const int per = stretch_of(seg[a.n_segments].at, gridDim.x);
    const int2 mine = pages_before(a, seg, blockIdx.x * per, (blockIdx.x + 1) * per);
    const int u0 = mine.x, u1 = mine.y;
    if (u0 >= u1) return;

    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem), q_base = (uint32_t)__cvta_generic_to_shared(q_s);
    constexpr int CK = D / 8, CV = kPageTokens / 8;        // 16-byte pieces of a row
    auto know = [&](int u) {        // pages u .. u + 31 into the ring
        if (tid < kBaKnown && u + tid < u1) ring[(u + tid - u0) % kBaRing] = unit_of(a, seg, lens, u + tid);
    };
    auto issue = [&](int u) {
        if (u < u1) {
            const Unit x = ring[(u - u0) % kBaRing];
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % STAGES) * T::kStage), vs = ks + kPageTokens * T::kPitchK;
            const __nv_bfloat16* k = (const __nv_bfloat16*)a.k_pool + (size_t)x.page * page_elements + head_off;
            const __nv_bfloat16* v = (const __nv_bfloat16*)a.v_pool + (size_t)x.page * page_elements + head_off;
            constexpr int RK = kBaThreads / CK, RV = kBaThreads / CV;
            if (x.keys == kPageTokens && kBaThreads % CK == 0 && RK % 8 == 0) {   // a thread's pieces lie whole rows apart, at one place in them
                const uint32_t kt = ks + T::k_piece(tid / CK, tid % CK), vt = vs + T::v_piece(tid / CV, tid % CV);
                k += tid * 8;
                v += tid * 8;
#pragma unroll
                for (int i = 0; i < kPageTokens / RK; ++i) cp_async16(kt + i * RK * T::kPitchK, k + i * kBaThreads * 8);
#pragma unroll
                for (int i = 0; i < D / RV; ++i) cp_async16(vt + i * RV * T::kPitchV, v + i * kBaThreads * 8);
            } else {
                for (int i = tid; i < kPageTokens * CK; i += kBaThreads)
                    cp_async16(ks + T::k_piece(i / CK, i % CK), k + (size_t)i * 8, i / CK < x.keys ? 16 : 0);
                // (values of positions past the sequence's end are read as zeros: a probability of 0 times what is not finite is not 0)
                for (int i = tid; i < D * CV; i += kBaThreads)
                    cp_async16(vs + T::v_piece(i / CV, i % CV), v + (size_t)i * 8, min(16, max(0, 2 * (x.keys - 8 * (i % CV)))));
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
    };
    know(u0);
    __syncthreads();
    int part_of = part_of_segment(a, ring[0].segment);
    if (!a.inv_freq) ask_queries(part_of);               // (they arrive with the first page)
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(u0 + i);
    if (a.inv_freq) ask_queries(part_of);                // (made while the first pages are on their way)

    const float scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    RowState<D> st;
    uint32_t qa[D / 16][4];
    int segment = -1, parts = 1, part = 0, tile = warp, rows = 0, lo_max = 0, row_end = 0, row_lo[2] = {0, 0};
    auto leave = [&](int u) {           // behind page u - 1, with its stage to join in
        const size_t piece = (size_t)kvh * (gridDim.x + a.n_segments) + blockIdx.x + segment;
        leave_tile<D>(st, reinterpret_cast<float*>(smem + ((u - 1 - u0) % STAGES) * T::kStage), parts, part, tile, lane, rows,
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
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) ldmatrix4(qa[ks], q_base + T::k_piece(row, ks * 2 + (lane >> 4)));
        }
        const int ahead = u + STAGES - 1;
        if (ahead < u1 && (ahead - u0) % kBaKnown == 0) {
            know(ahead);
            __syncthreads();
        }
        issue(ahead);
        if (a.write_cache && row_end - x.position <= kPageTokens) {      // a sequence's last page: its new key and value
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
            if (parts == 4) {
                attend_keys<D, 16>(st, qa, ks, vs, part * 16, lane, scale_log2, masked, x.position, row_lo, row_end);
            } else {
#pragma unroll 1
                for (int first = part * 32; first < kPageTokens; first += parts * 32)
                    attend_keys<D, 32>(st, qa, ks, vs, first, lane, scale_log2, masked, x.position, row_lo, row_end);
            }
        }
    }
    cp_async_wait<0>();
    leave(u1);
}

// float32, on multiply-adds.  Scores: a thread holds one key's dimensions in registers and takes every fourth row's query from shared memory
// (one broadcast for four multiply-adds); output: it holds one dimension's 64 values and takes the probabilities of its rows.  Sums are
// kept in four chains over the dimensions and four over the keys of a page, then a page's joins the row's.
constexpr int kBfThreads = 256;
template <int D>
struct BeamTileF32 {
    static constexpr int kPitchK = D + 4, kPitchV = kPageTokens + 4;       // floats: a multiple of 4, an odd number of 16 bytes
    static constexpr int kStage = kPageTokens * kPitchK + D * kPitchV;
    static constexpr int kStages = 2;
    static constexpr int kQ = kBaRows * kPitchK, kScores = kBaRows * kPitchV, kState = 3 * kBaRows;
    static constexpr int kBytes = 4 * (kStages * kStage + kQ + kScores + kState);
    static constexpr int kRowGroups = kBfThreads / D;                       // of the output: so many rows at a time
    static constexpr int kRowsEach = (kBaRows + kRowGroups - 1) / kRowGroups;
};

template <int D>
__global__ void __launch_bounds__(kBfThreads) attention_beams_f32_kernel(const __grid_constant__ BeamAttnArgs a) {
    using T = BeamTileF32<D>;
    extern __shared__ __align__(16) float smem_f[];
    __shared__ int tmp[kBfThreads / 16];
    __shared__ Unit ring[kBaRing];
    float* q_s = smem_f + T::kStages * T::kStage;
    float* p_s = q_s + T::kQ;                       // [row][kPitchV] scores, then probabilities
    float* m_s = p_s + T::kScores;
    float* l_s = m_s + kBaRows;
    float* f_s = l_s + kBaRows;                     // what a row's output so far is multiplied by
    Segment* seg = reinterpret_cast<Segment*>(f_s + kBaRows);
    int* lens = reinterpret_cast<int*>(seg + a.n_segments + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, rep = a.n_heads / a.n_kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    take_plan<kBfThreads>(a, seg, lens, tmp);
    const int per = stretch_of(seg[a.n_segments].at, gridDim.x);
    const int2 mine = pages_before(a, seg, blockIdx.x * per, (blockIdx.x + 1) * per);
    const int u0 = mine.x, u1 = mine.y;
    if (u0 >= u1) return;

    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem_f);
    auto know = [&](int u) {
        if (tid < kBaKnown && u + tid < u1) ring[(u + tid - u0) % kBaRing] = unit_of(a, seg, lens, u + tid);
    };
    auto issue = [&](int u) {
        if (u < u1) {
            const Unit x = ring[(u - u0) % kBaRing];
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % T::kStages) * T::kStage * 4), vs = ks + kPageTokens * T::kPitchK * 4;
            const float* k = (const float*)a.k_pool + (size_t)x.page * page_elements + head_off;
            const float* v = (const float*)a.v_pool + (size_t)x.page * page_elements + head_off;
            constexpr int CK = D / 4, CV = kPageTokens / 4;
#pragma unroll 4
            for (int i = tid; i < kPageTokens * CK; i += kBfThreads) {
                const int row = i / CK, c = i % CK;
                cp_async16(ks + (row * T::kPitchK + c * 4) * 4, k + (size_t)row * D + c * 4, row < x.keys ? 16 : 0);
            }
#pragma unroll 4
            for (int i = tid; i < D * CV; i += kBfThreads) {
                const int row = i / CV, c = i % CV;
                cp_async16(vs + (row * T::kPitchV + c * 4) * 4, v + (size_t)row * kPageTokens + c * 4, min(16, max(0, 4 * (x.keys - 4 * c))));
            }
        }
        cp_async_commit();
    };
    know(u0);
    __syncthreads();
    issue(u0);

    const float scale = 1.f / sqrtf((float)D);
    const int key = tid % kPageTokens, score_group = tid / kPageTokens;
    const int dim = tid % D, row_group = tid / D;
    float o[T::kRowsEach];
    int segment = -1, part_of = -1, rows = 0, q_row = 0, lo_max = 0, own_row = -1, r0 = 0;
    auto leave = [&]() {
        const size_t piece = (size_t)kvh * (gridDim.x + a.n_segments) + blockIdx.x + segment;
        float* to = a.part_o + piece * kBaRows * D;
        if (row_group < T::kRowGroups) {
#pragma unroll
            for (int j = 0; j < T::kRowsEach; ++j) {
                const int r = row_group + j * T::kRowGroups;
                if (r < rows) to[(size_t)r * D + dim] = o[j];
            }
        }
        for (int r = tid; r < rows; r += kBfThreads)
            *reinterpret_cast<float2*>(a.part_ml + (piece * kBaRows + r) * 2) = make_float2(m_s[r], l_s[r]);
    };
    for (int u = u0; u < u1; ++u) {
        cp_async_wait<0>();
        __syncthreads();
        const int ahead = u + 1;
        if (ahead < u1 && (ahead - u0) % kBaKnown == 0) {
            know(ahead);
            __syncthreads();
        }
        issue(ahead);
        const Unit x = ring[(u - u0) % kBaRing];
        if (x.segment != segment) {
            if (segment >= 0) leave();
            segment = x.segment;
#pragma unroll
            for (int j = 0; j < T::kRowsEach; ++j) o[j] = 0.f;
            const int p = part_of_segment(a, segment), i = segment - p * (a.sub_beams + 1), n = part_rows(a, p);
            r0 = part_first_row(a, p);
            __syncthreads();        // (the rows' m and l, and the queries, have been read)
            if (p != part_of) {
                part_of = p;
                constexpr int CQ = D / 4;
                for (int c = tid; c < n * rep * CQ; c += kBfThreads) {
                    const int row = c / CQ, at = c % CQ;
                    const float* from = (const float*)a.q + (size_t)(r0 + row / rep) * a.q_row_stride + (size_t)(kvh * rep + row % rep) * D + at * 4;
                    *reinterpret_cast<float4*>(q_s + row * T::kPitchK + at * 4) = *reinterpret_cast<const float4*>(from);
                }
            }
            rows = i == 0 ? n * rep : rep;
            q_row = i == 0 ? 0 : (i - 1) * rep;
            own_row = i == 0 ? -1 : r0 + i - 1;
            for (int r = tid; r < kBaRows; r += kBfThreads) { m_s[r] = -INFINITY; l_s[r] = 0.f; }
            lo_max = 0;
            if (i == 0) for (int b = 0; b < n; ++b) lo_max = max(lo_max, first_key(lens[r0 + b], a.window));
            else lo_max = first_key(lens[own_row], a.window);
            __syncthreads();
        }
        const float* k_tile = smem_f + ((u - u0) % T::kStages) * T::kStage;
        const float* v_tile = k_tile + kPageTokens * T::kPitchK;
        const bool masked = x.keys < kPageTokens || x.position < lo_max;
        {
            float4 k[D / 4];
#pragma unroll
            for (int c = 0; c < D / 4; ++c) k[c] = *reinterpret_cast<const float4*>(k_tile + key * T::kPitchK + c * 4);
            for (int r = score_group; r < rows; r += kBfThreads / kPageTokens) {
                const float* q = q_s + (q_row + r) * T::kPitchK;
                float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                for (int c = 0; c < D / 4; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(q + c * 4);
                    s0 += v.x * k[c].x; s1 += v.y * k[c].y; s2 += v.z * k[c].z; s3 += v.w * k[c].w;
                }
                float s = ((s0 + s1) + (s2 + s3)) * scale;
                if (masked) {
                    const int seq = own_row >= 0 ? own_row : r0 + r / rep, at = x.position + key;
                    if (key >= x.keys || at < first_key(lens[seq], a.window)) s = -INFINITY;
                }
                p_s[r * T::kPitchV + key] = s;
            }
        }
        __syncthreads();
        for (int r = warp; r < rows; r += kBfThreads / 32) {
            float* p = p_s + r * T::kPitchV;
            const float s0 = p[lane], s1 = p[lane + 32], m0 = m_s[r], m = fmaxf(m0, warp_max(fmaxf(s0, s1)));
            const float base = m == -INFINITY ? 0.f : m, e0 = expf(s0 - base), e1 = expf(s1 - base), sum = warp_sum(e0 + e1);
            p[lane] = e0;
            p[lane + 32] = e1;
            __syncwarp();
            if (lane == 0) {
                const float f = expf(m0 - base);
                f_s[r] = f;
                l_s[r] = l_s[r] * f + sum;
                m_s[r] = m;
            }
        }
        __syncthreads();
        if (row_group < T::kRowGroups) {
            float4 v[kPageTokens / 4];
#pragma unroll
            for (int c = 0; c < kPageTokens / 4; ++c) v[c] = *reinterpret_cast<const float4*>(v_tile + dim * T::kPitchV + c * 4);
#pragma unroll
            for (int j = 0; j < T::kRowsEach; ++j) {
                const int r = row_group + j * T::kRowGroups;
                if (r < rows) {
                    const float* p = p_s + r * T::kPitchV;
                    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                    for (int c = 0; c < kPageTokens / 4; ++c) {
                        const float4 w = *reinterpret_cast<const float4*>(p + c * 4);
                        s0 += w.x * v[c].x; s1 += w.y * v[c].y; s2 += w.z * v[c].z; s3 += w.w * v[c].w;
                    }
                    o[j] = o[j] * f_s[r] + ((s0 + s1) + (s2 + s3));
                }
            }
        }
    }
    leave();
}

// A warp per (sequence, query head): the pieces that hold the row, first those of the shared pages, then of its own.  A lane reads a piece's maximum
// and sum; the outputs are asked for eight pieces at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_beams_join_kernel(const __grid_constant__ BeamAttnArgs a, int n_ctas) {
    constexpr int E = D / 32, kAtOnce = 8;
    // maxima are in units of log 2 where the scores were, in bfloat16
    auto power = [](float x) { return sizeof(T) == 2 ? exp2_fast(x) : expf(x); };
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
        const int2 s0 = of[2 * shared], s1 = of[2 * shared + 2], o0 = of[2 * own], o1 = of[2 * own + 2], end = of[2 * a.n_segments];
        const unsigned per = (unsigned)stretch_of(end.y, n_ctas), magic = per > 1 ? 0xffffffffu / per + 1u : 0u;
        auto cta_of = [&](int x) {              // x / per
            if (magic == 0u) return x;
            const unsigned q = __umulhi((unsigned)x, magic);
            return (int)((unsigned long long)q * per > (unsigned)x ? q - 1u : q);
        };
        const int sa = s0.y + kSegmentCost, oa = o0.y + kSegmentCost, sn = s1.x - s0.x, on = o1.x - o0.x;
        c0 = cta_of(sa);
        n0 = sn > 0 ? cta_of(sa + sn - 1) - c0 + 1 : 0;
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
        const float top = fmaxf(m, warp_max(ml.x)), zero = top == -INFINITY ? 0.f : top, keep = power(m - zero), f = power(ml.x - zero);
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
                     int window) {
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
    return 0;
}

constexpr int kSmShared = 228 * 1024, kCtaShared = 227 * 1024, kCtaReserved = 1024;      // bytes of an SM, the most of a CTA's, what each takes besides

template <typename Kernel>
static int launch_beams(Kernel kernel, void (*join)(const BeamAttnArgs, int), int threads, int smem, int (&configured)[64], const BeamAttnArgs& a, int n_ctas,
                        cudaStream_t stream) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kErrBadArgument;
    if (configured[device] < smem) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        configured[device] = smem;
    }
    const int st = launch_pdl(kernel, dim3(n_ctas, a.n_kv_heads), dim3(threads), smem, stream, a);
    if (st != 0) return st;
    const long long rows = (long long)a.n_seqs * a.n_heads;
    return launch_pdl(join, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, a, n_ctas);
}

// bytes of dynamic shared memory with that many stages
template <int D>
static int beam_smem(const BeamAttnArgs& a, int stages) {
    return stages * BeamTile<D>::kStage + a.sub_beams * ((a.n_heads / a.n_kv_heads) * BeamTile<D>::kPitchK + (a.inv_freq ? D * 4 : 0)) + plan_ints(a) * 4;
}

template <int D>
static int launch_beams_of(int dtype, const BeamAttnArgs& a, int n_ctas, cudaStream_t stream) {
    static int configured[3][64] = {};
    const auto join = dtype == kBF16 ? attention_beams_join_kernel<__nv_bfloat16, D> : attention_beams_join_kernel<float, D>;
    if (dtype == kF32) {
        const int smem = BeamTileF32<D>::kBytes + plan_ints(a) * 4;
        if (smem + 2048 > kCtaShared) return kErrUnsupportedSize;
        return launch_beams(attention_beams_f32_kernel<D>, join, kBfThreads, smem, configured[0], a, n_ctas, stream);
    }
    // As many stages as leave room for three CTAs an SM with heads of up to 64, two with wider ones.
    constexpr int kMore = D <= 64 ? 4 : 3, kResident = D <= 64 ? 3 : 2, kStatic = 16 + kBaRing * (int)sizeof(Unit);
    const int smem = beam_smem<D>(a, kMore);
    if (smem + kStatic + kCtaReserved <= kSmShared / kResident)
        return launch_beams(attention_beams_kernel<D, kMore>, join, kBaThreads, smem, configured[1], a, n_ctas, stream);
    return launch_beams(attention_beams_kernel<D, 2>, join, kBaThreads, beam_smem<D>(a, 2), configured[2], a, n_ctas, stream);
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
                                         int n_kv_heads, int window, int fresh, cudaStream_t stream) {
    using namespace b200;
    if (n_groups <= 0) return 0;
    BeamAttnArgs a;
    const int st = fill_args(a, kv_lens, shared_pages, table_stride, n_groups, beams, n_heads, n_kv_heads, window);
    if (st != 0) return st;
    if (((uintptr_t)plan & 15) != 0) return kErrUnsupportedSize;
    a.plan = plan;
    a.fresh = fresh != 0;
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kErrBadArgument;
    const int smem = plan_ints(a) * 4;
    if (smem > 48 * 1024 && !configured[device]) {
        const cudaError_t e = cudaFuncSetAttribute(attention_beams_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCtaShared - 1024);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        configured[device] = true;
    }
    return launch_pdl(attention_beams_plan_kernel, dim3(1), dim3(256), smem, stream, a);
}

namespace b200 {

static int attention_beams(const void* q, long long q_row_stride, void* out, const int* kv_lens, const int* page_table, int table_stride,
                           const int* shared_pages, const void* k_pool, const void* v_pool, float* scratch, long long scratch_floats, int n_groups, int beams,
                           int n_heads, int n_kv_heads, int head_dim, int window, int n_parts, int dtype, const int* plan, const float* inv_freq, int pairing,
                           int write_cache, cudaStream_t stream) {
    if (n_groups <= 0) return 0;
    BeamAttnArgs a;
    const int st = fill_args(a, kv_lens, shared_pages, table_stride, n_groups, beams, n_heads, n_kv_heads, window);
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
