// A beam search's selection: of every request's beams and the whole vocabulary, the `keep` best continuations.
//
//   total[g, b, t] = scores[g, b] + (x[g, b, t] - lse[g, b]),   lse = m + log sum_t exp(x_t - m),   m = max_t x_t
//
// ordered by total, ties by the lower beam, then the larger logit, then the lower token.  Within a row the order of the totals
// is that of the logits, so each row's own best `keep` are found among the logits, without its lse; only those meet the
// other beams' on one scale.  Two launches:
//   beam_rows   a CTA per (chunk of a row, row): the chunk is read once, into registers, and leaves its maximum, its sum of
//               exponentials and its best `keep` logits in order;
//   beam_merge  a CTA per request: the rows' lse from their chunks' maxima and sums, the totals of what the chunks left, and
//               the best of those.
// Exponentials are taken in 32 bits and added in 32 bits over a thread's sixteen and a warp's lanes, from there on in 64: a
// row's lse is off by about 1e-8, and totals are compared in 64 bits, so that two beams' continuations change places only
// where they are that near to each other.  A score is rounded to 32 bits once, when it is stored.
//
// Rows that have no distribution give no candidates: a beam whose score is not finite (one that does not count, not read at
// all), a row that holds NaN or +inf, a row of nothing but -inf.  A logit of -inf is never a candidate.  Places for which there is
// none are stored as (-inf, -1, -1).
#include <limits.h>
#include "common.cuh"

namespace b200 {

constexpr int kBeamThreads = 256;                       // of beam_rows
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamEach = 16;                           // logits of a thread
constexpr int kBeamChunk = kBeamThreads * kBeamEach;    // logits of a CTA
constexpr int kBeamList = 512;                          // candidates that are ordered by counting
constexpr int kBeamMaxKeep = 256;
constexpr int kMergeThreads = 512;
constexpr int kMergeList = 1024;

// What a chunk leaves: [row][chunk] maximum (float) and sum (double), then [row][chunk][keep] logit and token, the best first, tokens of -1
// behind the last.
struct BeamScratch {
    double* sums;
    float* maxima;
    float* logits;
    int* tokens;
};
__host__ __device__ inline BeamScratch beam_scratch(void* base, long long pieces, int keep) {
    BeamScratch s;
    s.sums = (double*)base;
    s.maxima = (float*)(s.sums + pieces);
    s.logits = s.maxima + pieces;
    s.tokens = (int*)(s.logits + pieces * keep);
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

__global__ void __launch_bounds__(kBeamThreads)
beam_rows_kernel(const float* __restrict__ logits, long long ld, const float* __restrict__ scores, int vocab, int keep, int vec,
                 BeamScratch out) {
    __shared__ float warp_max_s[kBeamWarps], warp_sum_s[kBeamWarps];
    __shared__ unsigned warp_key_s[kBeamWarps];
    __shared__ float list_x[kBeamList];
    __shared__ int list_t[kBeamList];
    __shared__ int list_n;
    __shared__ unsigned long long warp_best_s[kBeamWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float score = scores[row];
    if (!(fabsf(score) < INFINITY)) return;     // (the merge does not look at this row either)
    const size_t piece = (size_t)row * gridDim.x + blockIdx.x;
    const int base = blockIdx.x * kBeamChunk, n = min(kBeamChunk, vocab - base);
    const float* x0 = logits + (size_t)row * ld + base;

    float x[kBeamEach];
    auto place = [&](int e) {       // of a thread's element e in the chunk
        return vec ? ((e >> 2) * kBeamThreads + tid) * 4 + (e & 3) : e * kBeamThreads + tid;
    };
    if (vec) {
#pragma unroll
        for (int u = 0; u < kBeamEach / 4; ++u) {
            const int at = (u * kBeamThreads + tid) * 4;
            if (at + 4 <= n) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(x0 + at));
                x[4 * u] = v.x; x[4 * u + 1] = v.y; x[4 * u + 2] = v.z; x[4 * u + 3] = v.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[4 * u + c] = at + c < n ? x0[at + c] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) x[e] = place(e) < n ? x0[place(e)] : -INFINITY;
    }
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < kBeamEach; ++e) { x[e] += 0.f; mine = fmaxf(mine, x[e]); }     // (-0 counts as 0)
    if (tid == 0) list_n = 0;

    // The warp's maximum and sum, and the j-th largest of its lanes' maxima: the warps' smallest such number is one that at
    // least warps * j >= keep logits reach, and few more than that do.
    const int j = (keep + kBeamWarps - 1) / kBeamWarps;
    unsigned key = rising_bits(mine), threshold = 0;
    float m = -INFINITY;
    if (j <= 32) {
        for (int i = 0; i < j; ++i) {
            threshold = __reduce_max_sync(0xffffffffu, key);
            if (i == 0) m = from_rising_bits(threshold);
            const unsigned at = __ballot_sync(0xffffffffu, key == threshold);
            if (lane == __ffs(at) - 1) key = 0;
        }
    }
    float sum = 0.f;
    if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) sum += expf(x[e] - m);
    } else {        // nothing but -inf, or NaN: which has to show
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) if (isnan(x[e])) sum = x[e];
    }
    sum = warp_sum(sum);
    if (lane == 0) {
        warp_max_s[warp] = m;
        warp_sum_s[warp] = sum;
        warp_key_s[warp] = threshold;
    }
    __syncthreads();
    unsigned least = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) least = min(least, warp_key_s[w]);
    least = max(least, kRisingMinusInf + 1u);           // -inf is no candidate
    if (tid == 0) {
        float top = -INFINITY;
        for (int w = 0; w < kBeamWarps; ++w) top = fmaxf(top, warp_max_s[w]);
        double total = 0.0;
        for (int w = 0; w < kBeamWarps; ++w) {
            const double s = (double)warp_sum_s[w];
            total += warp_max_s[w] > -INFINITY ? s * exp((double)warp_max_s[w] - (double)top) : s;
        }
        out.maxima[piece] = top;
        out.sums[piece] = total;
    }
    const float border = from_rising_bits(least);
#pragma unroll
    for (int e = 0; e < kBeamEach; ++e) {
        if (x[e] >= border) {
            const int i = atomicAdd(&list_n, 1);
            if (i < kBeamList) { list_x[i] = x[e]; list_t[i] = base + place(e); }
        }
    }
    __syncthreads();
    float* to_x = out.logits + piece * keep;
    int* to_t = out.tokens + piece * keep;
    const int found = list_n;
    if (found <= kBeamList) {
        // the list's order does not matter: every candidate's place is the number of those before it
        for (int i = tid; i < found; i += kBeamThreads) {
            const float v = list_x[i];
            const int t = list_t[i];
            int before = 0;
            for (int k = 0; k < found; ++k) before += (list_x[k] > v || (list_x[k] == v && list_t[k] < t)) ? 1 : 0;
            if (before < keep) { to_x[before] = v; to_t[before] = t; }
        }
        for (int i = found + tid; i < keep; i += kBeamThreads) to_t[i] = -1;
        return;
    }
    // Many logits reach the border (a chunk that is masked for the most part, or holds equal numbers): one after the other.
    for (int r = 0; r < keep; ++r) {
        unsigned long long best = 0;    // the rising bits, then the lower place
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) {
            const unsigned b = rising_bits(x[e]);
            if (x[e] > -INFINITY) best = max(best, ((unsigned long long)b << 32) | (unsigned)(0xffffffffu - place(e)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) warp_best_s[warp] = best;
        __syncthreads();
        best = warp_best_s[0];
#pragma unroll
        for (int w = 1; w < kBeamWarps; ++w) best = max(best, warp_best_s[w]);
        __syncthreads();
        const int at = (int)(0xffffffffu - (unsigned)best);
        if (tid == 0) {
            to_x[r] = best ? from_rising_bits((unsigned)(best >> 32)) : -INFINITY;
            to_t[r] = best ? base + at : -1;
        }
        if (best) {
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) if (place(e) == at) x[e] = -INFINITY;
        }
    }
}

struct Candidate {
    double total;
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

__global__ void __launch_bounds__(kMergeThreads)
beam_merge_kernel(const float* __restrict__ scores, int beams, int chunks, int keep, BeamScratch in, float* __restrict__ out_scores,
                  int* __restrict__ out_beams, int* __restrict__ out_tokens) {
    __shared__ double list_total[kMergeList];
    __shared__ float list_logit[kMergeList];
    __shared__ int list_beam[kMergeList], list_token[kMergeList];
    __shared__ int list_n;
    __shared__ unsigned warp_key_s[kMergeThreads / 32];
    __shared__ Candidate warp_best_s[kMergeThreads / 32];
    extern __shared__ double lse_s[];       // [beams]; NaN: the row gives none
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kMergeThreads / 32;
    if (tid == 0) list_n = 0;
    pdl_launch_dependents();
    pdl_wait();
    for (int b = warp; b < beams; b += kWarps) {
        const size_t row = (size_t)g * beams + b;
        const float score = scores[row];
        double lse = NAN;
        if (fabsf(score) < INFINITY) {
            float top = -INFINITY;
            for (int c = lane; c < chunks; c += 32) top = fmaxf(top, in.maxima[row * chunks + c]);
            top = warp_max(top);
            double total = 0.0;
            for (int c = lane; c < chunks; c += 32) {
                const float mc = in.maxima[row * chunks + c];
                const double s = in.sums[row * chunks + c];
                total += mc > -INFINITY ? s * exp((double)mc - (double)top) : s;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            lse = top > -INFINITY && top < INFINITY && total < (double)INFINITY ? (double)top + log(total) : NAN;    // (a NaN sum gives NaN)
        }
        if (lane == 0) lse_s[b] = lse;
    }
    __syncthreads();

    const int lists = beams * chunks;       // in the order of beams
    const size_t first_list = (size_t)g * lists;
    auto candidate = [&](int list, int k) {
        Candidate c{-INFINITY, -INFINITY, 0, -1};
        if (list >= lists || k >= keep) return c;
        const int b = list / chunks;
        const double lse = lse_s[b];
        if (isnan(lse)) return c;
        const size_t at = (first_list + list) * keep + k;
        c.token = in.tokens[at];
        if (c.token < 0) return c;
        c.logit = in.logits[at];
        c.beam = b;
        c.total = (double)scores[(size_t)g * beams + b] + ((double)c.logit - lse);
        return c;
    };

    // As in beam_rows: of every warp's lists the j-th best head, rounded down to 32 bits; at least `keep` candidates reach the least of them.
    const int used_warps = min(kWarps, (lists + 31) / 32), j = (keep + used_warps - 1) / used_warps;
    unsigned key = 0, threshold = 0;
    for (int l = tid; l < lists; l += kMergeThreads) {
        const Candidate c = candidate(l, 0);
        if (c.token >= 0) key = max(key, rising_bits(__double2float_rd(c.total)));
    }
    if (j <= 32) {
        for (int i = 0; i < j; ++i) {
            threshold = __reduce_max_sync(0xffffffffu, key);
            const unsigned at = __ballot_sync(0xffffffffu, key == threshold);
            if (lane == __ffs(at) - 1) key = 0;
        }
    }
    if (lane == 0) warp_key_s[warp] = threshold;
    __syncthreads();
    unsigned least = 0xffffffffu;
    for (int w = 0; w < used_warps; ++w) least = min(least, warp_key_s[w]);
    for (int l = tid; l < lists; l += kMergeThreads) {
        for (int k = 0; k < keep; ++k) {
            const Candidate c = candidate(l, k);
            if (c.token < 0 || rising_bits(__double2float_rd(c.total)) < least) break;
            const int i = atomicAdd(&list_n, 1);
            if (i < kMergeList) { list_total[i] = c.total; list_logit[i] = c.logit; list_beam[i] = c.beam; list_token[i] = c.token; }
        }
    }
    __syncthreads();
    const size_t to = (size_t)g * keep;
    const int found = list_n;
    if (found <= kMergeList) {
        for (int i = tid; i < found; i += kMergeThreads) {
            const Candidate c{list_total[i], list_logit[i], list_beam[i], list_token[i]};
            int before = 0;
            for (int k = 0; k < found; ++k) {
                const double o = list_total[k];
                if (o > c.total) ++before;
                else if (o == c.total) before += goes_before(Candidate{o, list_logit[k], list_beam[k], list_token[k]}, c) ? 1 : 0;
            }
            if (before < keep) {
                out_scores[to + before] = (float)c.total;
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
    Candidate last{INFINITY, INFINITY, -1, INT_MAX};
    for (int r = 0; r < keep; ++r) {
        Candidate best{-INFINITY, -INFINITY, 0, -1};
        for (int l = tid; l < lists; l += kMergeThreads) {
            for (int k = 0; k < keep; ++k) {
                const Candidate c = candidate(l, k);
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
        if (lane == 0) warp_best_s[warp] = best;
        __syncthreads();
        best = warp_best_s[0];
        for (int w = 1; w < kWarps; ++w) if (goes_before(warp_best_s[w], best)) best = warp_best_s[w];
        __syncthreads();
        last = best;
        if (tid == 0) {
            out_scores[to + r] = best.token >= 0 ? (float)best.total : -INFINITY;
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

// Bytes of scratch (16-byte aligned) that a call needs.
extern "C" long long b200_beam_select_scratch_bytes(int n_rows, int vocab, int keep) {
    const long long pieces = (long long)n_rows * ((vocab + b200::kBeamChunk - 1) / b200::kBeamChunk);
    return pieces * (12 + 8ll * keep);
}

// logits: [n_groups * beams] rows of `vocab` floats, `ld` apart; scores: [n_groups, beams]; outputs: [n_groups, keep].
extern "C" int b200_beam_select(const float* logits, long long ld, const float* scores, float* out_scores, int* out_beams, int* out_tokens,
                                void* scratch, long long scratch_bytes, int n_groups, int beams, int vocab, int keep, cudaStream_t stream) {
    using namespace b200;
    if (n_groups <= 0) return 0;
    if (beams < 1 || vocab < 1 || keep < 1 || ld < vocab) return kErrBadArgument;
    if (keep > kBeamMaxKeep || beams > 1024 || (long long)n_groups * beams > 65535) return kErrUnsupportedSize;
    const int chunks = (vocab + kBeamChunk - 1) / kBeamChunk;
    const long long rows = (long long)n_groups * beams;
    if (scratch_bytes < b200_beam_select_scratch_bytes((int)rows, vocab, keep)) return 10003;
    const BeamScratch s = beam_scratch(scratch, rows * chunks, keep);
    const int vec = ((uintptr_t)logits & 15) == 0 && (ld & 3) == 0;
    const int st = launch_pdl(beam_rows_kernel, dim3(chunks, (unsigned)rows), dim3(kBeamThreads), 0, stream, logits, ld, scores, vocab, keep,
                              vec, s);
    if (st != 0) return st;
    return launch_pdl(beam_merge_kernel, dim3(n_groups), dim3(kMergeThreads), sizeof(double) * beams, stream, scores, beams, chunks, keep, s,
                      out_scores, out_beams, out_tokens);
}
