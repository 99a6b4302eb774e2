// A beam search's selection: of every request's beams and the whole vocabulary, the `keep` best continuations.
//
//   total[g, b, t] = scores[g, b] + (x[g, b, t] - m) - log sum_t exp(x_t - m),   m = max_t x_t
//
// ordered by total, ties by the lower beam, then the larger logit, then the lower token.  Within a row the order of the totals
// is that of the logits, so each row's own best `keep` are found among the logits, without its lse; only those meet the
// other beams' on one scale.  Two launches:
//   beam_rows   a CTA per (chunk of a row, row): the chunk is read once, in tiles of 4,096 logits, and leaves a sum of
//               exponentials with what they are relative to and its best `keep` logits in order;
//   beam_merge  a CTA per request: the rows' lse from their chunks' maxima and sums, the totals of what the chunks left, and
//               the best of those.
//
// beam_rows keeps one list of candidates a CTA: logits that reach a border.  The border is first what about `keep` of the threads' maxima
// of the first tile reach, so that few logits beyond `keep` are ever listed, and rises when the list is cut down; a thread of a later tile
// compares its sixteen logits' maximum once and mostly goes on.  So a chunk costs the reading, an exponential a logit, and a few
// searches of 32 steps with a barrier each.  (Lists of each warp by itself need no barriers, but then every warp holds `keep`
// candidates of its own and the ordering at the end is of eight times as many, which took longer than all the rest.)
//
// Exponentials are taken in 32 bits, relative to a whole number that no logit so far exceeds by more than 1, added in 32 bits over eight of a
// thread's logits and in 64 from there on.  In units of 2^-24 an exponential of x - m = -t is off by 2.3 t (the difference, the product with log2 e,
// that number's rounding) and 4 (the power of two), the additions by 8; weighed by the probabilities t is at most 1 + log V.  So a row's lse is off by
// at most 2^-24 (2.3 (1 + log V) + 12), 2.5e-6 for 128,256 tokens (absolutely; measured, the selected scores of ordinary rows, -20 or so, are off by 2.7e-8
// of their norm, their own rounding included).  Totals are compared in 64 bits, so two beams' continuations change places only where they are that near to each other, and
// none is above its beam's score, whatever the lse is off by.  A score is rounded to 32 bits once, when it is stored.
//
// Bound by: HBM in bytes (4 per logit), in fact by the rows' instructions and the merge's chain of barriers.  Measured: 64 rows of
// 128,256 logits, 16 kept each of 8, 18.3 us of which the reading needs 5.0; 256 rows, 64 kept, 47.8 us of 20.0 (rows 39 us at 3.4 TB/s,
// issuing in half of all cycles); 4 rows 10.5 us, of which the two launches, the first tile's search and the merge are nearly all.
//
// Rows that have no distribution give no candidates: a beam whose score is not finite (one that does not count, not read at
// all), a row that holds NaN or +inf, a row of nothing but -inf.  A logit of -inf is never a candidate.  Places for which there is
// none are stored as (-inf, -1, -1).
#include <limits.h>
#include "common.cuh"

namespace b200 {

constexpr int kBeamThreads = 256;                       // of beam_rows
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamEach = 16;                           // logits of a thread at a time
constexpr int kBeamTile = kBeamThreads * kBeamEach;
constexpr int kBeamMaxKeep = 256;
constexpr int kBeamLimit = kBeamMaxKeep + kBeamMaxKeep / 2 + 32;      // most candidates of a list that is not cut down
constexpr int kBeamList = kBeamLimit + kBeamTile;       // most that it holds
constexpr int kMergeThreads = 512;
constexpr int kMergeList = 1024;

typedef unsigned long long u64;

// What a chunk leaves: [row][chunk] a sum of exponentials and what they are relative to, [row][chunk][keep] candidates, the best first, zeros behind
// the last.
struct BeamScratch {
    double* sums;
    u64* candidates;
    float* maxima;
};
__host__ __device__ inline BeamScratch beam_scratch(void* base, long long pieces, int keep) {
    BeamScratch s;
    s.sums = (double*)base;
    s.candidates = (u64*)(s.sums + pieces);
    s.maxima = (float*)(s.candidates + pieces * keep);
    return s;
}

// Unsigned numbers that rise with the float (0: below every number that is not NaN).
__device__ __forceinline__ unsigned rising_bits(float x) {
    const unsigned b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_rising_bits(unsigned r) {
    return __uint_as_float((r & 0x80000000u) ? r & 0x7fffffffu : ~r);
}
constexpr unsigned kRisingMinusInf = 0x007fffffu;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A candidate as one number: a larger logit, of equal ones a lower token, is the larger number.
__device__ __forceinline__ u64 beam_key(float x, int token) { return ((u64)rising_bits(x) << 32) | (0xffffffffu - (unsigned)token); }
__device__ __forceinline__ float key_logit(u64 key) { return from_rising_bits((unsigned)(key >> 32)); }
__device__ __forceinline__ int key_token(u64 key) { return (int)(0xffffffffu - (unsigned)key); }

// Exponentials are taken relative to whole numbers, so that what stands between two sums is a power e^-n, looked up in 64 bits (whose functions take
// longer than all the rest of a merge); beyond 63 it is below what a sum in 64 bits keeps of the larger one's rounding in 32.
__constant__ double kPowers[64] = {
    1.00000000000000000e+00, 3.67879441171442334e-01, 1.35335283236612702e-01, 4.97870683678639445e-02, 1.83156388887341787e-02, 6.73794699908546700e-03,
    2.47875217666635849e-03, 9.11881965554516244e-04, 3.35462627902511853e-04, 1.23409804086679561e-04, 4.53999297624848542e-05, 1.67017007902456593e-05,
    6.14421235332820981e-06, 2.26032940698105424e-06, 8.31528719103567877e-07, 3.05902320501825786e-07, 1.12535174719259116e-07, 4.13993771878516683e-08,
    1.52299797447126292e-08, 5.60279643753726783e-09, 2.06115362243855787e-09, 7.58256042791190660e-10, 2.78946809286892464e-10, 1.02618796317018902e-10,
    3.77513454427909773e-11, 1.38879438649640209e-11, 5.10908902806332510e-12, 1.87952881653908324e-12, 6.91440010694020302e-13, 2.54366564737692275e-13,
    9.35762296884017482e-14, 3.44247710846997675e-14, 1.26641655490941755e-14, 4.65888614510339774e-15, 1.71390843154201300e-15, 6.30511676014698922e-16,
    2.31952283024356963e-16, 8.53304762574406580e-17, 3.13913279204802960e-17, 1.15482241730157861e-17, 4.24835425529158887e-18, 1.56288218933498879e-18,
    5.74952226429355990e-19, 2.11513103759108046e-19, 7.78113224113379661e-20, 2.86251858054939366e-20, 1.05306173575538117e-20, 3.87399762868718678e-21,
    1.42516408274093515e-21, 5.24288566336346390e-22, 1.92874984796391782e-22, 7.09547416228470366e-23, 2.61027906966770474e-23, 9.60268005450867556e-24,
    3.53262857220080711e-24, 1.29958142500750312e-24, 4.78089288388546882e-25, 1.75879220242431161e-25, 6.47023492564545988e-26, 2.38026640869440067e-26,
    8.75651076269652004e-27, 3.22134028599251593e-27, 1.18506486423398097e-27, 4.35961000006308085e-28,
};
__device__ __forceinline__ double brought_to(double sum, float from, float to) {     // from <= to, whole numbers or -inf (a sum of 0, or NaN)
    const float n = to - from;
    return n < 64.f ? sum * kPowers[(int)n] : (n >= 64.f && !isnan(sum) ? 0.0 : sum);
}

struct RowsShared {
    u64 list[kBeamList];                // 36 KB
    int n;
    float ref[kBeamWarps];
    double sum[kBeamWarps];
    int count[2][kBeamWarps];
    unsigned high[kBeamWarps], low[kBeamWarps];
};

// Cuts the CTA's list (more than `keep` candidates) down to its best, at least `keep` and at most a quarter more.  What they reach is
// searched for bit by bit, candidates of equal logits by their tokens.  Returns its upper half.  All threads call it, behind a barrier.
__device__ __forceinline__ unsigned cut_down(RowsShared& sh, int keep) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = sh.n;
    int round = 0;
    auto total = [&](int mine) {
        mine = __reduce_add_sync(0xffffffffu, mine);
        round ^= 1;                     // (two sets of counts in turn: one barrier a count)
        if (lane == 0) sh.count[round][warp] = mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kBeamWarps; ++w) all += sh.count[round][w];
        return all;
    };
    // (the bits that all candidates have in common are not searched)
    unsigned high = 0, low = 0xffffffffu;
    for (int i = tid; i < n; i += kBeamThreads) {
        high = max(high, (unsigned)(sh.list[i] >> 32));
        low = min(low, (unsigned)(sh.list[i] >> 32));
    }
    high = __reduce_max_sync(0xffffffffu, high);
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) { sh.high[warp] = high; sh.low[warp] = low; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) { high = max(high, sh.high[w]); low = min(low, sh.low[w]); }
    const int differing = 32 - __clz(high ^ low);
    if (n <= kBeamThreads) {            // one candidate a thread: it stays in a register, and a barrier counts
        const u64 key = tid < n ? sh.list[tid] : 0ull;
        u64 least = differing == 32 ? 0ull : ((u64)high << 32) >> (32 + differing) << (32 + differing);
        for (int bit = 31 + differing; bit >= 0; --bit) {
            const u64 t = least | (1ull << bit);
            const int reach = __syncthreads_count(key >= t);
            if (reach >= keep) {
                least = t;
                if (reach <= keep + keep / 4) break;
            }
        }
        if (tid == 0) sh.n = 0;
        __syncthreads();
        if (key >= least && key != 0ull) sh.list[atomicAdd(&sh.n, 1)] = key;
        __syncthreads();
        return (unsigned)(least >> 32);
    }
    u64 least = differing == 32 ? 0ull : ((u64)high << 32) >> (32 + differing) << (32 + differing);
    for (int bit = 31 + differing; bit >= 0; --bit) {
        const u64 t = least | (1ull << bit);
        int mine = 0;
        for (int i = tid; i < n; i += kBeamThreads) mine += sh.list[i] >= t ? 1 : 0;
        mine = total(mine);
        if (mine >= keep) {
            least = t;
            if (mine <= keep + keep / 4) break;
        }
    }
    // in place, a stretch of 256 after the other: nothing goes behind where it was
    int kept = 0;
    for (int i0 = 0; i0 < n; i0 += kBeamThreads) {
        const u64 key = i0 + tid < n ? sh.list[i0 + tid] : 0ull;
        const bool in = key >= least && key != 0ull;
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        round ^= 1;
        if (lane == 0) sh.count[round][warp] = __popc(mask);
        __syncthreads();
        int at = kept;
#pragma unroll
        for (int w = 0; w < kBeamWarps; ++w) {
            if (w < warp) at += sh.count[round][w];
            kept += sh.count[round][w];
        }
        if (in) sh.list[at + __popc(mask & ((1u << lane) - 1u))] = key;
    }
    if (tid == 0) sh.n = kept;
    __syncthreads();
    return (unsigned)(least >> 32);
}

__global__ void __launch_bounds__(kBeamThreads, 4)
beam_rows_kernel(const float* __restrict__ logits, long long ld, const float* __restrict__ scores, int vocab, int keep, int vec, int tiles,
                 BeamScratch out) {
    __shared__ RowsShared sh;
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sh.n = 0;
    pdl_launch_dependents();
    pdl_wait();
    const float score = scores[row];
    if (!(fabsf(score) < INFINITY)) return;     // (the merge does not look at this row either)
    const size_t piece = (size_t)row * gridDim.x + blockIdx.x;
    const int first = blockIdx.x * tiles * kBeamTile, end = min(vocab, first + tiles * kBeamTile);
    const float* x_row = logits + (size_t)row * ld;

    auto place = [&](int e) { return vec ? ((e >> 2) * kBeamThreads + tid) * 4 + (e & 3) : e * kBeamThreads + tid; };    // in a tile
    auto load = [&](float (&x)[kBeamEach], int base) {
        const int n = end - base;
        const float* x0 = x_row + base;
        if (vec && n >= kBeamTile) {
#pragma unroll
            for (int u = 0; u < kBeamEach / 4; ++u) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(x0) + u * kBeamThreads + tid);
                x[4 * u] = v.x; x[4 * u + 1] = v.y; x[4 * u + 2] = v.z; x[4 * u + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) x[e] = place(e) < n ? __ldg(x0 + place(e)) : -INFINITY;
        }
    };
    const int limit = max(128, keep + keep / 2 + 32);
    float border = 0.f;         // what candidates reach
    float ref = -INFINITY;      // the thread's exponentials are relative to it
    double total = 0.0;
    float x[kBeamEach], ahead[kBeamEach];
    load(ahead, first);
    for (int base = first; base < end; base += kBeamTile) {
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) x[e] = ahead[e];
        if (base + kBeamTile < end) load(ahead, base + kBeamTile);
        float mine = x[0];
#pragma unroll
        for (int e = 1; e < kBeamEach; ++e) mine = fmaxf(mine, x[e]);

        if (base == first) {
            // What about the keep-th largest of the threads' maxima reach, at least `keep` logits do, and few more.
            const unsigned key = isnan(mine) ? 0u : rising_bits(mine), top = __reduce_max_sync(0xffffffffu, key);
            ref = top ? ceilf(from_rising_bits(top)) : -INFINITY;
            unsigned least = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned t = least | (1u << bit);
                const int n = __syncthreads_count(key >= t);
                if (n >= keep) {
                    least = t;
                    if (n <= keep + keep / 4) break;
                }
            }
            border = from_rising_bits(max(least, kRisingMinusInf + 1u));     // -inf is no candidate
        }
        if (mine > ref + 1.f) {         // (relative to the maximum of the warp's first logits until that is exceeded)
            const float higher = ceilf(mine);
            total = ref > -INFINITY ? brought_to(total, ref, higher) : total;
            ref = higher;
        }
        const float zero = ref == -INFINITY ? 0.f : ref;     // (nothing but -inf so far, or NaN, which has to show)
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) sum[e & 1] += exp2_fast((x[e] - zero) * 1.4426950408889634f);
        total += (double)(sum[0] + sum[1]);

        int reached = 0;            // the list's length behind this thread's candidates
        if (mine >= border) {
            unsigned hits = 0;
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) hits |= x[e] >= border ? 1u << e : 0u;
            int at = atomicAdd(&sh.n, __popc(hits));
            reached = at + __popc(hits);
            for (; hits; hits &= hits - 1) {
                const int e = __ffs(hits) - 1;
                float v = x[0];
#pragma unroll
                for (int k = 1; k < kBeamEach; ++k) v = e == k ? x[k] : v;
                sh.list[at++] = beam_key(v + 0.f, base + place(e));      // (-0 counts as 0)
            }
        }
        // (the barrier itself says whether the list is too long: sh.n, read behind it, may be the next tile's already, whose first threads do not wait)
        if (__syncthreads_or(reached > limit)) border = fmaxf(border, from_rising_bits(cut_down(sh, keep)));
    }
    {
        const float r = warp_max(ref);
        if (ref < r && ref > -INFINITY) total = brought_to(total, ref, r);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) { sh.ref[warp] = r; sh.sum[warp] = total; }
    }
    __syncthreads();
    if (sh.n > 128 && sh.n > keep) cut_down(sh, keep);
    if (warp == 0) {
        const float w = lane < kBeamWarps ? sh.ref[lane] : -INFINITY, r = warp_max(w);
        double t = lane < kBeamWarps ? sh.sum[lane] : 0.0;
        if (w < r && w > -INFINITY) t = brought_to(t, w, r);
#pragma unroll
        for (int o = kBeamWarps / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) { out.maxima[piece] = r; out.sums[piece] = t; }
    }
    // in order: every candidate's place is the number of those before it
    const int found = sh.n;
    u64* to = out.candidates + piece * keep;
    for (int i0 = 0; i0 < found; i0 += kBeamThreads / 4) {      // four threads a candidate
        const int i = i0 + (tid >> 2);
        const u64 key = i < found ? sh.list[i] : ~0ull;
        int before = 0;
        for (int k = tid & 3; k < found; k += 4) before += sh.list[k] > key ? 1 : 0;
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        if (i < found && before < keep && (tid & 3) == 0) to[before] = key;
    }
    for (int i = found + tid; i < keep; i += kBeamThreads) to[i] = 0ull;
}

struct Candidate {
    u64 total;              // a number that rises with it
    float logit;
    int beam, token;        // token -1: none
};
__device__ __forceinline__ bool goes_before(const Candidate& a, const Candidate& b) {
    if (b.token < 0) return a.token >= 0;
    if (a.token < 0) return false;
    if (a.total != b.total) return a.total > b.total;
    if (a.beam != b.beam) return a.beam < b.beam;
    if (a.logit != b.logit) return a.logit > b.logit;
    return a.token < b.token;
}
__device__ __forceinline__ u64 rising_bits(double x) {
    const u64 b = (u64)__double_as_longlong(x + 0.0);
    return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double double_of(u64 r) { return __longlong_as_double((long long)((r >> 63) ? r & ~(1ull << 63) : ~r)); }

constexpr int kMergeEach = 8, kMergeKeys = kMergeEach * kMergeThreads;
constexpr int kMergeWarps = kMergeThreads / 32;
struct MergeShared {
    u64 keys[kMergeKeys];               // rough total and number of candidates
    u64 total[kMergeList];
    float logit[kMergeList];
    int beam[kMergeList], token[kMergeList];
    int active[kMergeList];             // lists that may hold some of the best
    Candidate warp_best[kMergeWarps];
    int count[2][kMergeWarps];
    unsigned high[kMergeWarps];
    int n_keys, n_active, n;
    unsigned largest;                   // of the beams' |base|, its bits
};
struct Beam {
    double exact;       // score - log of the row's sum of exponentials (NaN: the row gives none)
    float ref;          // what the sum is relative to
    float base;         // the first, rounded
    float score;        // which no total exceeds
};

// 64-bit arithmetic is slow on this chip (a comparison of 80 by 80 totals took 8 us), so candidates are found by rough totals in 32 bits, off by
// at most half a step of each of their three parts, with a border lowered by more than that; exact totals are made of those that
// reach it, about as many as are wanted, and are put in order as whole numbers.
__global__ void __launch_bounds__(kMergeThreads)
beam_merge_kernel(const float* __restrict__ scores, int beams, int chunks, int keep, BeamScratch in, float* __restrict__ out_scores,
                  int* __restrict__ out_beams, int* __restrict__ out_tokens) {
    extern __shared__ __align__(16) unsigned char merge_smem[];
    MergeShared& sh = *reinterpret_cast<MergeShared*>(merge_smem);
    Beam* beam_s = reinterpret_cast<Beam*>(merge_smem + sizeof(MergeShared));
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) { sh.n = sh.n_active = sh.n_keys = 0; sh.largest = 0; }
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();            // (sh.largest grows below)
    const int lists = beams * chunks;       // in the order of beams
    const long long all = (long long)lists * keep;
    const u64* from = in.candidates + (size_t)g * all;
    // where all candidates fit the threads' registers they are asked for before anything else
    const bool at_once = all <= kMergeKeys;
    const unsigned chunks_magic = 0xffffffffu / (unsigned)chunks + 1u, keep_magic = 0xffffffffu / (unsigned)keep + 1u;      // 2^32 / d, rounded up
    u64 held[kMergeEach];
    if (at_once) {
#pragma unroll
        for (int u = 0; u < kMergeEach; ++u) held[u] = tid + u * kMergeThreads < all ? from[tid + u * kMergeThreads] : 0ull;
    }
    for (int b = warp; b < beams; b += kMergeWarps) {
        const size_t row = ((size_t)g * beams + b) * chunks;
        const float score = scores[(size_t)g * beams + b];
        double base = NAN;
        float top = -INFINITY;
        if (fabsf(score) < INFINITY) {          // (nothing was left for other rows)
            for (int c = lane; c < chunks; c += 32) top = fmaxf(top, in.maxima[row + c]);
            top = warp_max(top);
            double total = 0.0;
            for (int c = lane; c < chunks; c += 32) {
                const float mc = in.maxima[row + c];
                const double s = in.sums[row + c];
                total += mc > -INFINITY && mc < top ? brought_to(s, mc, top) : s;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            // (a NaN sum gives NaN)
            if (top > -INFINITY && top < INFINITY && total < (double)INFINITY) base = (double)score - log(total);
        }
        if (lane == 0) {
            beam_s[b] = Beam{base, top, (float)base, score};
            if (!isnan(base)) atomicMax(&sh.largest, __float_as_uint(fabsf((float)base)));
        }
    }
    __syncthreads();

    auto beam_of = [&](int list) { return chunks == 1 ? list : (int)__umulhi((unsigned)list, chunks_magic); };       // (exact below 2^16)
    auto list_of = [&](unsigned number) { return at_once ? (keep == 1 ? (int)number : (int)__umulhi(number, keep_magic)) : (int)(number / keep); };
    auto key_at = [&](int list, int k) { return list < lists && k < keep ? from[(size_t)list * keep + k] : 0ull; };
    // a candidate's rough total, as a number that rises with it; 0: none
    auto rough = [&](u64 key, int list) {
        if (key == 0ull) return 0u;
        const Beam& b = beam_s[beam_of(list)];
        const float t = (key_logit(key) - b.ref) + b.base;
        return isnan(t) ? 0u : rising_bits(fminf(t, b.score) + 0.f);
    };
    auto exact = [&](u64 key, int list) {
        Candidate c{0ull, -INFINITY, 0, -1};
        if (key == 0ull) return c;
        c.beam = beam_of(list);
        const Beam& b = beam_s[c.beam];
        if (isnan(b.base)) return c;
        c.token = key_token(key);
        c.logit = key_logit(key);
        // (the log sum may be off by so much that a token of probability 1 comes out above its beam's score)
        c.total = rising_bits(fmin(((double)c.logit - (double)b.ref) + b.exact, (double)b.score));
        return c;
    };
    // what is taken when `least` is what enough rough totals reach: everything that may be exactly as large
    auto lowered = [&](unsigned least) {
        const float t = from_rising_bits(least);
        return max(rising_bits(t - 4.8e-7f * (fabsf(t) + __uint_as_float(sh.largest))), 1u);      // (8 half steps of either)
    };
    // The largest number that `need` of all threads' keys reach (0: there are not as many), or one that few more do; `mine`: the thread's largest.  What
    // lies above the largest of all, and the bits that numbers between it and the least of the warps' largest have in common, are not searched where
    // those are enough already.
    auto search = [&](auto count_mine, unsigned mine, int need) {
        mine = __reduce_max_sync(0xffffffffu, mine);
        if (lane == 0) sh.high[warp] = mine;
        __syncthreads();
        const unsigned w = lane < kMergeWarps ? sh.high[lane] : 0u, high = __reduce_max_sync(0xffffffffu, w);
        int set = 0;
        auto reaching = [&](unsigned t) {
            int n = __reduce_add_sync(0xffffffffu, count_mine(t));
            set ^= 1;               // (two sets of counts in turn, call by call, whichever bits are counted: one barrier a count)
            if (lane == 0) sh.count[set][warp] = n;
            __syncthreads();
            return (int)__reduce_add_sync(0xffffffffu, lane < kMergeWarps ? sh.count[set][lane] : 0);
        };
        // numbers that differ from the largest in their last 24 bits only: totals within a factor of four or so
        unsigned least = high & 0xff000000u;
        int bit = 23;
        if (reaching(least) < need) { least = 0; bit = 31; }
        for (; bit >= 0; --bit) {
            const unsigned t = least | (1u << bit);
            const int n = t <= high ? reaching(t) : 0;
            if (n >= need) {
                least = t;
                if (n <= need + need / 4) break;
            }
        }
        return least ? lowered(least) : 1u;
    };
    unsigned least = 1;
    bool listed = true;         // what may be among the best has gone to the list
    u64 mine[kMergeEach];       // rough total and number
    if (at_once) {
#pragma unroll
        for (int u = 0; u < kMergeEach; ++u) {
            const int i = tid + u * kMergeThreads;
            mine[u] = ((u64)rough(held[u], list_of(i)) << 32) | (unsigned)i;
        }
    } else {
        // A number that at least `keep` candidates reach and not many more: where there are lists enough, one that `keep` of the threads'
        // best heads reach; where there are few, one that so many of their (depth + 1)-th best reach that it comes to as much.
        bool head = false;
        for (int l = tid; l < lists; l += kMergeThreads) head = head || rough(key_at(l, 0), l) != 0u;
        const int n_heads = __syncthreads_count(head);
        const int depth = n_heads >= keep || n_heads == 0 ? 0 : (2 * keep + n_heads - 1) / n_heads - 1;
        unsigned key = 0;
        for (int l = tid; l < lists; l += kMergeThreads) key = max(key, rough(key_at(l, depth), l));
        least = search([&](unsigned t) { return key >= t ? 1 : 0; }, key, (keep + depth) / (depth + 1));
        __syncthreads();
        // the lists with a candidate that reaches it, a thread each; then of those, a warp each, all that reach it
        for (int l = tid; l < lists; l += kMergeThreads) {
            if (rough(key_at(l, 0), l) >= least) {
                const int i = atomicAdd(&sh.n_active, 1);
                if (i < kMergeList) sh.active[i] = l;
            }
        }
        __syncthreads();
        const int n_active = sh.n_active;
        for (int a = warp; a < min(n_active, kMergeList); a += kMergeWarps) {
            for (int k0 = 0; k0 < keep; k0 += 32) {
                const unsigned b = rough(key_at(sh.active[a], k0 + lane), sh.active[a]);
                const bool in = b >= least;
                if (in) {
                    const int i = atomicAdd(&sh.n_keys, 1);
                    if (i < kMergeKeys) sh.keys[i] = ((u64)b << 32) | (unsigned)(sh.active[a] * keep + k0 + lane);
                }
                if (!__any_sync(0xffffffffu, in)) break;
            }
        }
        __syncthreads();
        listed = n_active <= kMergeList && sh.n_keys <= kMergeKeys;
#pragma unroll
        for (int u = 0; u < kMergeEach; ++u) mine[u] = tid + u * kMergeThreads < min(sh.n_keys, kMergeKeys) ? sh.keys[tid + u * kMergeThreads] : 0ull;
    }
    if (listed) {
        unsigned best = 0;
#pragma unroll
        for (int u = 0; u < kMergeEach; ++u) best = max(best, (unsigned)(mine[u] >> 32));
        least = search([&](unsigned t) {
            int n = 0;
#pragma unroll
            for (int u = 0; u < kMergeEach; ++u) n += (unsigned)(mine[u] >> 32) >= t ? 1 : 0;
            return n;
        }, best, keep);
#pragma unroll
        for (int u = 0; u < kMergeEach; ++u) {
            if ((unsigned)(mine[u] >> 32) >= least) {
                const unsigned number = (unsigned)mine[u];
                const Candidate c = exact(at_once ? held[u] : from[number], list_of(number));
                const int i = atomicAdd(&sh.n, 1);
                if (i < kMergeList) { sh.total[i] = c.total; sh.logit[i] = c.logit; sh.beam[i] = c.beam; sh.token[i] = c.token; }
            }
        }
    }
    __syncthreads();
    const size_t to = (size_t)g * keep;
    const int found = listed ? sh.n : kMergeList + 1;
    if (found <= kMergeList) {
        for (int i0 = 0; i0 < found; i0 += kMergeThreads / 4) {         // four threads a candidate
            const int i = i0 + (tid >> 2), at = min(i, found - 1);
            const Candidate c{sh.total[at], sh.logit[at], sh.beam[at], sh.token[at]};
            int before = 0;
            for (int k = tid & 3; k < found; k += 4) {
                const u64 o = sh.total[k];
                before += o > c.total ? 1 : 0;
                if (o == c.total && k != at) before += goes_before(Candidate{o, sh.logit[k], sh.beam[k], sh.token[k]}, c) ? 1 : 0;
            }
            before += __shfl_xor_sync(0xffffffffu, before, 1);
            before += __shfl_xor_sync(0xffffffffu, before, 2);
            if (i < found && before < keep && (tid & 3) == 0) {
                out_scores[to + before] = (float)double_of(c.total);
                out_beams[to + before] = c.beam;
                out_tokens[to + before] = c.token;
            }
        }
        for (int i = found + tid; i < keep; i += kMergeThreads) {
            out_scores[to + i] = -INFINITY;
            out_beams[to + i] = -1;
            out_tokens[to + i] = -1;
        }
        return;
    }
    // More than the list holds reach the border (many equal totals): the best head of all lists, `keep` times.  What a thread has
    // taken from its lists is found again by the order: it hands out what comes behind the last one taken from all.
    Candidate last{~0ull, INFINITY, -1, INT_MAX};
    for (int r = 0; r < keep; ++r) {
        Candidate best{0ull, -INFINITY, 0, -1};
        for (int l = tid; l < lists; l += kMergeThreads) {
            for (int k = 0; k < keep; ++k) {
                const Candidate c = exact(key_at(l, k), l);
                if (c.token < 0) break;
                if (r > 0 && !goes_before(last, c)) continue;
                if (goes_before(c, best)) best = c;
                break;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Candidate c;
            c.total = __shfl_xor_sync(0xffffffffu, best.total, o);
            c.logit = __shfl_xor_sync(0xffffffffu, best.logit, o);
            c.beam = __shfl_xor_sync(0xffffffffu, best.beam, o);
            c.token = __shfl_xor_sync(0xffffffffu, best.token, o);
            if (goes_before(c, best)) best = c;
        }
        if (lane == 0) sh.warp_best[warp] = best;
        __syncthreads();
        best = sh.warp_best[0];
        for (int w = 1; w < kMergeWarps; ++w) if (goes_before(sh.warp_best[w], best)) best = sh.warp_best[w];
        __syncthreads();
        last = best;
        if (tid == 0) {
            out_scores[to + r] = best.token >= 0 ? (float)double_of(best.total) : -INFINITY;
            out_beams[to + r] = best.token >= 0 ? best.beam : -1;
            out_tokens[to + r] = best.token;
        }
        if (best.token < 0) {
            for (int i = r + 1 + tid; i < keep; i += kMergeThreads) {
                out_scores[to + i] = -INFINITY;
                out_beams[to + i] = -1;
                out_tokens[to + i] = -1;
            }
            return;
        }
    }
}

}  // namespace b200

namespace b200 {
// Tiles of a CTA: so many that all rows' CTAs are on the GPU at once, four an SM; the tiles behind the first meet a border that few of
// their logits reach, and the merge has fewer lists.  Rows beyond that are a CTA each.
static int tiles_of(long long rows, int vocab) {
    const long long tiles = (vocab + kBeamTile - 1) / kBeamTile, ctas = 4ll * device_sm_count() / rows;
    return (int)(ctas < 1 ? tiles : (tiles + ctas - 1) / ctas);
}
}  // namespace b200

// Bytes of scratch (16-byte aligned) that a call needs.
extern "C" long long b200_beam_select_scratch_bytes(int n_rows, int vocab, int keep) {
    const int chunk = b200::tiles_of(n_rows, vocab) * b200::kBeamTile;
    return (long long)n_rows * ((vocab + chunk - 1) / chunk) * (12 + 8ll * keep);
}

// logits: [n_groups * beams] rows of `vocab` floats, `ld` apart; scores: [n_groups, beams]; outputs: [n_groups, keep].
extern "C" int b200_beam_select(const float* logits, long long ld, const float* scores, float* out_scores, int* out_beams, int* out_tokens,
                                void* scratch, long long scratch_bytes, int n_groups, int beams, int vocab, int keep, cudaStream_t stream) {
    using namespace b200;
    if (n_groups <= 0) return 0;
    if (beams < 1 || vocab < 1 || keep < 1 || ld < vocab) return kErrBadArgument;
    if (keep > kBeamMaxKeep || beams > 1024 || vocab > (1 << 30) || (long long)n_groups * beams > 65535) return kErrUnsupportedSize;
    const long long rows = (long long)n_groups * beams;
    const int tiles = tiles_of(rows, vocab), chunks = (vocab + tiles * kBeamTile - 1) / (tiles * kBeamTile);
    if (scratch_bytes < b200_beam_select_scratch_bytes((int)rows, vocab, keep)) return 10003;
    const BeamScratch s = beam_scratch(scratch, rows * chunks, keep);
    const int vec = ((uintptr_t)logits & 15) == 0 && (ld & 3) == 0;
    const size_t merge_bytes = sizeof(MergeShared) + sizeof(Beam) * beams;
    static bool configured[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kErrBadArgument;
    if (!configured[device]) {
        const cudaError_t e = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(MergeShared) + sizeof(Beam) * 1024));
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        configured[device] = true;
    }
    const int st = launch_pdl(beam_rows_kernel, dim3(chunks, (unsigned)rows), dim3(kBeamThreads), 0, stream, logits, ld, scores, vocab, keep,
                              vec, tiles, s);
    if (st != 0) return st;
    return launch_pdl(beam_merge_kernel, dim3(n_groups), dim3(kMergeThreads), merge_bytes, stream, scores, beams, chunks, keep, s,
                      out_scores, out_beams, out_tokens);
}
