// One decode step's attention of sequences that come in groups (the beams of a request) and share their first pages.
//
//   o[r, h] = softmax_j(q[r, h] . k[j, h / rep] / sqrt(D)) v[j, h / rep],   j < kv_len[r]  (with a window: j >= kv_len[r] - window)
//
// Groups are `beams` consecutive sequences; the first shared_pages[g] entries of their page-table rows name the same pages, all of
// them full.  Those are read once for all beams of the group and all query heads of a kv head, which are the rows of one
// tile: at 8 beams of 32 heads on 8 that is 32 rows, and an eighth of the bytes that as many separate sequences read.
//
// The work is cut by pages.  The pages of one segment belong together: the shared pages of a group, then the pages that each
// of its sequences has for itself, group after group.  All segments' pages in this order are numbered, and of every kv head each of
// gridDim.x CTAs takes as many consecutive ones, whatever they belong to, so groups of unequal length share the GPU evenly.
// A CTA keeps the running maximum m, sum l and output o of a segment's rows in registers and leaves them, unnormalised, in
// scratch at the segment's end or its own; a second kernel joins what the CTAs left of a row, in a fixed order.  CTA c's piece of
// segment s is number c + s (along the pages either grows, so no two pieces have one number).
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
    int* plan;                          // [0] pages of a CTA, [1 + s] first page number of segment s, of which the last is the end
    long long q_row_stride;
    int table_stride, n_seqs, n_groups, beams, sub_beams, n_sub, n_heads, n_kv_heads, window;
};

__device__ __forceinline__ int first_key(int kv_len, int window) { return window > 0 ? max(0, kv_len - window) : 0; }

// Segments: part p of n_groups * n_sub (n_sub parts of up to sub_beams sequences to a group) has its shared pages as segment p * (sub_beams + 1),
// its sequences' own as the next ones.
__device__ __forceinline__ int part_first_row(const BeamAttnArgs& a, int p) { return (p / a.n_sub) * a.beams + (p % a.n_sub) * a.sub_beams; }
__device__ __forceinline__ int part_rows(const BeamAttnArgs& a, int p) { return min(a.sub_beams, a.beams - (p % a.n_sub) * a.sub_beams); }
// the shared pages [lo, hi) that some sequence of the part reads; hi bounds the sequences' own pages from below
__device__ __forceinline__ void shared_range(const BeamAttnArgs& a, int p, int& lo, int& hi) {
    const int r0 = part_first_row(a, p), n = part_rows(a, p);
    hi = min(max(a.shared_pages[p / a.n_sub], 0), a.table_stride);
    int first = 0x7fffffff;
    for (int i = 0; i < n; ++i) {
        const int len = max(a.kv_lens[r0 + i], 0);
        hi = min(hi, len / kPageTokens);
        first = min(first, first_key(len, a.window));
    }
    lo = min(first / kPageTokens, hi);
}
__device__ __forceinline__ void own_range(const BeamAttnArgs& a, int row, int shared_hi, int& lo, int& hi) {
    const int len = max(a.kv_lens[row], 0);
    hi = min((len + kPageTokens - 1) / kPageTokens, a.table_stride);
    lo = min(max(shared_hi, first_key(len, a.window) / kPageTokens), hi);
}

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, int bytes) {      // the rest of the 16 is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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

// A page of the work: whose it is, where, and how much of it holds keys.
struct Unit {
    int page, segment, position, keys;
};

// The plan, by all threads of a CTA: seg_s[s] = number of pages before segment s, seg_s[n_segments] = all.  `tmp`: an int for each warp.
template <int THREADS>
__device__ __forceinline__ void make_plan(const BeamAttnArgs& a, int n_segments, int* seg_s, int* tmp) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_part = a.sub_beams + 1;
    // a thread's consecutive segments, their pages first counted, then added up in order
    const int each = (n_segments + THREADS - 1) / THREADS, s0 = tid * each, s1 = min(n_segments, s0 + each);
    int total = 0;
    for (int s = s0; s < s1; ++s) {
        const int p = s / per_part, i = s % per_part;
        int lo, hi, n = 0;
        shared_range(a, p, lo, hi);
        if (i == 0) n = hi - lo;
        else if (i <= part_rows(a, p)) {
            own_range(a, part_first_row(a, p) + i - 1, hi, lo, hi);
            n = hi - lo;
        }
        seg_s[s] = n;
        total += n;
    }
    int incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) tmp[warp] = incl;
    __syncthreads();
    int before = incl - total;
    for (int w = 0; w < warp; ++w) before += tmp[w];
    for (int s = s0; s < s1; ++s) {
        const int n = seg_s[s];
        seg_s[s] = before;
        before += n;
    }
    if (tid == THREADS - 1) seg_s[n_segments] = before;
    __syncthreads();
}

// the last segment that starts at or before page number u (and is not empty, u being one of its pages)
__device__ __forceinline__ int segment_of(const int* seg_s, int n_segments, int u) {
    int lo = 0, hi = n_segments - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seg_s[mid] <= u) lo = mid; else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ Unit unit_of(const BeamAttnArgs& a, const int* seg_s, int n_segments, int u) {
    Unit x;
    x.segment = segment_of(seg_s, n_segments, u);
    const int per_part = a.sub_beams + 1, p = x.segment / per_part, i = x.segment % per_part;
    int lo, hi;
    shared_range(a, p, lo, hi);
    const int r0 = part_first_row(a, p), row = i == 0 ? r0 : r0 + i - 1;
    if (i > 0) own_range(a, row, hi, lo, hi);
    const int index = lo + u - seg_s[x.segment];
    x.page = a.page_table[(size_t)row * a.table_stride + index];
    x.position = index * kPageTokens;
    x.keys = i == 0 ? kPageTokens : min(kPageTokens, a.kv_lens[row] - x.position);
    return x;
}

// bfloat16, on mma.sync.  A warp owns a tile of 16 rows and, where there are fewer than four tiles, a part of each page's keys.
template <int D>
struct BeamTile {
    static constexpr int kPitchK = 2 * D + 16, kPitchV = 2 * kPageTokens + 16;  // bytes; an odd number of 16: ldmatrix meets no bank twice
    static constexpr int kStage = kPageTokens * kPitchK + D * kPitchV;
    static constexpr int kStages = D <= 64 ? 3 : 2;
    static constexpr int kQ = kBaRows * kPitchK;
    static constexpr int kJoin = 2 * 16 * (D + 4) * 4;                          // two tiles' o, m, l
    static constexpr int kBytes = kStages * kStage + kQ + kJoin;
};

template <int D>
struct RowState {
    float o[D / 8][4];
    float m[2], l[2];               // of rows g and g + 8; l is a lane's share
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
};

// One page's keys [part * 64 / KP, ...) for the tile whose query fragments' rows start at q_addr (this lane's ldmatrix address).
template <int D, int KP>
__device__ __forceinline__ void attend_page(RowState<D>& st, uint32_t q_addr, uint32_t k_base, uint32_t v_base, int part, int lane, float scale_log2,
                                            bool masked, int position, const int (&row_lo)[2], int row_end) {
    constexpr int NK = kPageTokens / KP, NT = NK / 8;
    using T = BeamTile<D>;
    const int t = lane & 3;
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][c] = 0.f;
    // ldmatrix: lanes 0-7, 8-15, 16-23, 24-31 give the rows of the four 8 x 8 blocks (keys 0-7 and 8-15 by 8 dimensions and the next 8)
    const uint32_t k_lane = k_base + (uint32_t)((part * NK + (lane & 7) + (lane >> 4) * 8) * T::kPitchK + ((lane >> 3) & 1) * 16);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t qa[4];
        ldmatrix4(qa, q_addr + ks * 32);
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
            uint32_t kb[4];
            ldmatrix4(kb, k_lane + (uint32_t)(i * 8 * T::kPitchK + ks * 32));
            mma_bf16(s[i], qa, kb[0], kb[1]);
            mma_bf16(s[i + 1], qa, kb[2], kb[3]);
        }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            s[i][c] *= scale_log2;
            if (masked) {
                const int key = position + part * NK + 8 * i + 2 * t + (c & 1);
                if (key < row_lo[c >> 1] || key >= row_end) s[i][c] = -INFINITY;
            }
            top[c >> 1] = fmaxf(top[c >> 1], s[i][c]);
        }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        const float m = fmaxf(st.m[h], top[h]);
        const float base = m == -INFINITY ? 0.f : m;        // (a row that has seen nothing yet: its probabilities are 0)
        const float keep = exp2_fast(st.m[h] - base);
        st.m[h] = m;
        st.l[h] *= keep;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) { st.o[j][2 * h] *= keep; st.o[j][2 * h + 1] *= keep; }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float p = exp2_fast(s[i][2 * h + e] - base);
                st.l[h] += p;
                s[i][2 * h + e] = p;
            }
    }
    const uint32_t v_lane = v_base + (uint32_t)(((lane & 7) + (lane >> 4) * 8) * T::kPitchV + (part * NK + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
    for (int kk = 0; kk < NK / 16; ++kk) {
        // probabilities are rounded to bfloat16 for the tensor cores, as the values are stored; their sum l is not
        const uint32_t pa[4] = {pack2(s[2 * kk][0], s[2 * kk][1]), pack2(s[2 * kk][2], s[2 * kk][3]),
                                pack2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
            uint32_t vb[4];
            ldmatrix4(vb, v_lane + (uint32_t)(j * 8 * T::kPitchV + kk * 32));
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
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 1);
        st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 2);
    }
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
                if (t == 0) { row[D] = st.m[h]; row[D + 1] = st.l[h]; }
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
                st.l[h] = st.l[h] * c1 + l2 * c2;
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
        if (t == 0) *reinterpret_cast<float2*>(to_ml + 2 * r) = make_float2(st.m[h], st.l[h]);
    }
}

template <int D>
__global__ void __launch_bounds__(kBaThreads) attention_beams_kernel(const __grid_constant__ BeamAttnArgs a, int n_segments) {
    using T = BeamTile<D>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int tmp[kBaThreads / 32];
    __shared__ Unit ring[kBaRing];
    unsigned char* q_s = smem + T::kStages * T::kStage;
    float* join = reinterpret_cast<float*>(q_s + T::kQ);
    int* seg_s = reinterpret_cast<int*>(q_s + T::kQ + T::kJoin);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, rep = a.n_heads / a.n_kv_heads, per_part = a.sub_beams + 1;
    pdl_launch_dependents();
    pdl_wait();
    make_plan<kBaThreads>(a, n_segments, seg_s, tmp);
    const int all = seg_s[n_segments], per = max(1, (all + (int)gridDim.x - 1) / (int)gridDim.x);
    if (blockIdx.x == 0 && kvh == 0) {      // for the kernel that joins the pieces
        for (int s = tid; s <= n_segments; s += kBaThreads) a.plan[1 + s] = seg_s[s];
        if (tid == 0) a.plan[0] = per;
    }
    const int u0 = blockIdx.x * per, u1 = min(all, u0 + per);
    if (u0 >= u1) return;

    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem), q_base = (uint32_t)__cvta_generic_to_shared(q_s);
    auto know = [&](int u) {        // pages u .. u + 31 into the ring
        if (tid < kBaKnown && u + tid < u1) ring[(u + tid - u0) % kBaRing] = unit_of(a, seg_s, n_segments, u + tid);
    };
    auto issue = [&](int u) {
        if (u < u1) {
            const Unit x = ring[(u - u0) % kBaRing];
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % T::kStages) * T::kStage), vs = ks + kPageTokens * T::kPitchK;
            const __nv_bfloat16* k = (const __nv_bfloat16*)a.k_pool + (size_t)x.page * page_elements + head_off;
            const __nv_bfloat16* v = (const __nv_bfloat16*)a.v_pool + (size_t)x.page * page_elements + head_off;
            constexpr int CK = D / 8, CV = kPageTokens / 8;        // 16-byte pieces of a row
#pragma unroll
            for (int i = tid; i < kPageTokens * CK; i += kBaThreads) {
                const int row = i / CK, c = i % CK;
                cp_async16(ks + row * T::kPitchK + c * 16, k + (size_t)row * D + c * 8, row < x.keys ? 16 : 0);
            }
            // (values of positions past the sequence's end are read as zeros: a probability of 0 times what is not finite is not 0)
#pragma unroll
            for (int i = tid; i < D * CV; i += kBaThreads) {
                const int row = i / CV, c = i % CV;
                cp_async16(vs + row * T::kPitchV + c * 16, v + (size_t)row * kPageTokens + c * 8, min(16, max(0, 2 * (x.keys - 8 * c))));
            }
        }
        cp_async_commit();
    };
    know(u0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::kStages - 1; ++i) issue(u0 + i);

    const float scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    RowState<D> st;
    int segment = -1, part_of = -1, parts = 1, part = 0, tile = warp, rows = 0, q_row = 0, lo_max = 0, row_end = 0, row_lo[2] = {0, 0};
    auto leave = [&]() {
        const size_t piece = (size_t)kvh * (gridDim.x + n_segments) + blockIdx.x + segment;
        leave_tile<D>(st, join, parts, part, tile, lane, rows, a.part_o + piece * kBaRows * D, a.part_ml + piece * kBaRows * 2);
    };
    for (int u = u0; u < u1; ++u) {
        cp_async_wait<T::kStages - 2>();
        __syncthreads();
        const int ahead = u + T::kStages - 1;
        if (ahead < u1 && ahead > u0 && (ahead - u0) % kBaKnown == 0) {
            know(ahead);
            __syncthreads();
        }
        issue(ahead);
        const Unit x = ring[(u - u0) % kBaRing];
        if (x.segment != segment) {
            if (segment >= 0) leave();
            segment = x.segment;
            st.clear();
            const int p = segment / per_part, i = segment % per_part;
            const int r0 = part_first_row(a, p), n = part_rows(a, p);
            if (p != part_of) {         // the queries of all of the part's rows
                __syncthreads();
                part_of = p;
                constexpr int CQ = D / 8;
                for (int c = tid; c < n * rep * CQ; c += kBaThreads) {
                    const int row = c / CQ, at = c % CQ;
                    const __nv_bfloat16* from = (const __nv_bfloat16*)a.q + (size_t)(r0 + row / rep) * a.q_row_stride
                                                + (size_t)(kvh * rep + row % rep) * D + at * 8;
                    *reinterpret_cast<uint4*>(q_s + row * T::kPitchK + at * 16) = *reinterpret_cast<const uint4*>(from);
                }
                __syncthreads();
            }
            rows = i == 0 ? n * rep : rep;
            q_row = i == 0 ? 0 : (i - 1) * rep;
            const int tiles = (rows + 15) / 16;
            parts = tiles == 1 ? 4 : tiles == 2 ? 2 : 1;
            tile = warp % (4 / parts);
            part = warp / (4 / parts);
            lo_max = 0;
            if (i == 0) {
                for (int b = 0; b < n; ++b) lo_max = max(lo_max, first_key(a.kv_lens[r0 + b], a.window));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = min(tile * 16 + (lane >> 2) + 8 * h, rows - 1);
                    row_lo[h] = first_key(a.kv_lens[r0 + r / rep], a.window);
                }
                row_end = 0x7fffffff;
            } else {
                row_end = a.kv_lens[r0 + i - 1];
                lo_max = row_lo[0] = row_lo[1] = first_key(row_end, a.window);
            }
        }
        if (tile * 16 < rows) {
            // (rows behind the last one are its copies, and nothing of them is stored)
            const int row = min(tile * 16 + (lane & 15), rows - 1) + q_row;
            const uint32_t q_addr = q_base + (uint32_t)(row * T::kPitchK + (lane >> 4) * 16);
            const uint32_t ks = stage0 + (uint32_t)(((u - u0) % T::kStages) * T::kStage), vs = ks + kPageTokens * T::kPitchK;
            const bool masked = x.keys < kPageTokens || x.position < lo_max;
            if (parts == 4) attend_page<D, 4>(st, q_addr, ks, vs, part, lane, scale_log2, masked, x.position, row_lo, row_end);
            else if (parts == 2) attend_page<D, 2>(st, q_addr, ks, vs, part, lane, scale_log2, masked, x.position, row_lo, row_end);
            else attend_page<D, 1>(st, q_addr, ks, vs, part, lane, scale_log2, masked, x.position, row_lo, row_end);
        }
    }
    leave();
    cp_async_wait<0>();
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
__global__ void __launch_bounds__(kBfThreads) attention_beams_f32_kernel(const __grid_constant__ BeamAttnArgs a, int n_segments) {
    using T = BeamTileF32<D>;
    extern __shared__ __align__(16) float smem_f[];
    __shared__ int tmp[kBfThreads / 32];
    __shared__ Unit ring[kBaRing];
    float* q_s = smem_f + T::kStages * T::kStage;
    float* p_s = q_s + T::kQ;                       // [row][kPitchV] scores, then probabilities
    float* m_s = p_s + T::kScores;
    float* l_s = m_s + kBaRows;
    float* f_s = l_s + kBaRows;                     // what a row's output so far is multiplied by
    int* seg_s = reinterpret_cast<int*>(f_s + kBaRows);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, rep = a.n_heads / a.n_kv_heads, per_part = a.sub_beams + 1;
    pdl_launch_dependents();
    pdl_wait();
    make_plan<kBfThreads>(a, n_segments, seg_s, tmp);
    const int all = seg_s[n_segments], per = max(1, (all + (int)gridDim.x - 1) / (int)gridDim.x);
    if (blockIdx.x == 0 && kvh == 0) {
        for (int s = tid; s <= n_segments; s += kBfThreads) a.plan[1 + s] = seg_s[s];
        if (tid == 0) a.plan[0] = per;
    }
    const int u0 = blockIdx.x * per, u1 = min(all, u0 + per);
    if (u0 >= u1) return;

    const size_t page_elements = (size_t)a.n_kv_heads * kPageTokens * D, head_off = (size_t)kvh * kPageTokens * D;
    const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem_f);
    auto know = [&](int u) {
        if (tid < kBaKnown && u + tid < u1) ring[(u + tid - u0) % kBaRing] = unit_of(a, seg_s, n_segments, u + tid);
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
        const size_t piece = (size_t)kvh * (gridDim.x + n_segments) + blockIdx.x + segment;
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
            const int p = segment / per_part, i = segment % per_part, n = part_rows(a, p);
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
            if (i == 0) for (int b = 0; b < n; ++b) lo_max = max(lo_max, first_key(a.kv_lens[r0 + b], a.window));
            else lo_max = first_key(a.kv_lens[own_row], a.window);
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
                    if (key >= x.keys || at < first_key(a.kv_lens[seq], a.window)) s = -INFINITY;
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

// A warp per (sequence, query head): the pieces that hold the row, first those of the shared pages, then of its own.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_beams_join_kernel(const __grid_constant__ BeamAttnArgs a, int n_segments, int n_ctas) {
    constexpr int E = D / 32;
    // maxima are in units of log 2 where the scores were, in bfloat16
    auto power = [](float x) { return sizeof(T) == 2 ? exp2f(x) : expf(x); };
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (at >= (long long)a.n_seqs * a.n_heads) return;
    const int seq = (int)(at / a.n_heads), head = (int)(at % a.n_heads), rep = a.n_heads / a.n_kv_heads, kvh = head / rep;
    const int g = seq / a.beams, beam = seq % a.beams, p = g * a.n_sub + beam / a.sub_beams, i = beam % a.sub_beams;
    const int s = p * (a.sub_beams + 1), per = a.plan[0];
    const size_t base = (size_t)kvh * (n_ctas + n_segments);
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
    for (int own = 0; own < 2; ++own) {
        const int segment = own ? s + 1 + i : s, row = own ? head % rep : i * rep + head % rep;
        const int first = a.plan[1 + segment], end = a.plan[2 + segment];
        if (first >= end) continue;
        const int c0 = first / per, c1 = (end - 1) / per;
        for (int c = c0; c <= c1; c += 4) {
            float mc[4], lc[4], oc[4][E];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const size_t piece = (base + min(c + k, c1) + segment) * kBaRows + row;
                const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * piece);
                mc[k] = c + k <= c1 ? ml.x : -INFINITY;
                lc[k] = c + k <= c1 ? ml.y : 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) oc[k][e] = a.part_o[piece * D + e * 32 + lane];
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, mc[k]);
            const float zero = top == -INFINITY ? 0.f : top, keep = power(m - zero);
            l *= keep;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= keep;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = power(mc[k] - zero);
                l += lc[k] * f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += f > 0.f ? oc[k][e] * f : 0.f;
            }
            m = top;
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
    return (segments + n_parts) * n_kv_heads * kBaRows * (head_dim + 2) + ((segments + 2 + 3) / 4) * 4;
}

template <typename Kernel>
static int launch_beams(Kernel kernel, void (*join)(const BeamAttnArgs, int, int), int threads, int smem, int (&configured)[64], const BeamAttnArgs& a,
                        int n_segments, int n_parts, cudaStream_t stream) {
    smem += (n_segments + 1) * 4;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kErrBadArgument;
    if (configured[device] < smem) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        configured[device] = smem;
    }
    const int st = launch_pdl(kernel, dim3(n_parts, a.n_kv_heads), dim3(threads), smem, stream, a, n_segments);
    if (st != 0) return st;
    const long long rows = (long long)a.n_seqs * a.n_heads;
    return launch_pdl(join, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, a, n_segments, n_parts);
}

template <int D>
static int launch_beams_of(int dtype, const BeamAttnArgs& a, int n_segments, int n_parts, cudaStream_t stream) {
    static int configured[64] = {}, configured_f32[64] = {};
    if (dtype == kBF16)
        return launch_beams(attention_beams_kernel<D>, attention_beams_join_kernel<__nv_bfloat16, D>, kBaThreads, BeamTile<D>::kBytes, configured, a,
                            n_segments, n_parts, stream);
    return launch_beams(attention_beams_f32_kernel<D>, attention_beams_join_kernel<float, D>, kBfThreads, BeamTileF32<D>::kBytes, configured_f32, a,
                        n_segments, n_parts, stream);
}

}  // namespace b200

extern "C" long long b200_attention_beams_scratch_floats(int n_groups, int beams, int n_heads, int n_kv_heads, int head_dim, int n_parts) {
    if (n_groups < 1 || beams < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads / n_kv_heads > b200::kBaRows) return 0;
    return b200::scratch_floats_of(n_groups, beams, n_heads, n_kv_heads, head_dim, n_parts);
}

// Sequences are n_groups groups of `beams`; kv_lens[n_seqs], page_table [n_seqs][table_stride], shared_pages[n_groups].  n_parts: CTAs of
// a kv head.  Keys and values of the step are in the cache already.
extern "C" int b200_attention_beams(const void* q, long long q_row_stride, void* out, const int* kv_lens, const int* page_table, int table_stride,
                                    const int* shared_pages, const void* k_pool, const void* v_pool, float* scratch, long long scratch_floats,
                                    int n_groups, int beams, int n_heads, int n_kv_heads, int head_dim, int window, int n_parts,
                                    int dtype, cudaStream_t stream) {
    using namespace b200;
    if (n_groups <= 0) return 0;
    if ((dtype != kF32 && dtype != kBF16) || beams < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || window < 0 || n_parts < 1 || table_stride < 1) return kErrBadArgument;
    const int rep = n_heads / n_kv_heads;
    if (rep > 16 || head_dim % 32 != 0 || head_dim < 32 || head_dim > 128 || n_kv_heads > 65535 || n_parts > 65535) return kErrUnsupportedSize;
    const long long segments = segments_of(n_groups, beams, rep);
    if (segments > kBaMaxSegments) return kErrUnsupportedSize;
    if (q_row_stride % (dtype == kBF16 ? 8 : 4) != 0 || (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch) & 15) != 0) return kErrUnsupportedSize;
    if (scratch_floats < scratch_floats_of(n_groups, beams, n_heads, n_kv_heads, head_dim, n_parts)) return 10003;
    BeamAttnArgs a;
    a.q = q; a.out = out; a.kv_lens = kv_lens; a.page_table = page_table; a.shared_pages = shared_pages; a.k_pool = k_pool; a.v_pool = v_pool;
    const long long pieces = (segments + n_parts) * n_kv_heads;
    a.part_o = scratch;
    a.part_ml = scratch + pieces * kBaRows * head_dim;
    a.plan = (int*)(a.part_ml + pieces * kBaRows * 2);
    a.q_row_stride = q_row_stride;
    a.table_stride = table_stride; a.n_seqs = n_groups * beams; a.n_groups = n_groups; a.beams = beams;
    a.sub_beams = beams_of_part(beams, rep);
    a.n_sub = (beams + a.sub_beams - 1) / a.sub_beams;
    a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.window = window;
    switch (head_dim) {
        case 32: return launch_beams_of<32>(dtype, a, (int)segments, n_parts, stream);
        case 64: return launch_beams_of<64>(dtype, a, (int)segments, n_parts, stream);
        case 96: return launch_beams_of<96>(dtype, a, (int)segments, n_parts, stream);
        default: return launch_beams_of<128>(dtype, a, (int)segments, n_parts, stream);
    }
}
