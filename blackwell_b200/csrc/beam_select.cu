// Beam search's selection: of the candidates  score[b] + log_softmax(logits[b])[v]  of a request's beams the best few.
//
// Two launches.  The first reads the logits once, a chunk of a row per block: the chunk's maximum and sum of exponentials, and its
// `keep` largest logits (within a row the order of the candidates is that of the logits).  The second, a block per request, forms the
// rows' log-sums and compares the chunks' candidates across the beams.  Log-sums, scores and comparisons are in 64 bits: two beams'
// candidates may lie closer to each other than 32 bits tell apart.
//
// Both find the best K of n values without sorting: the n values are dealt to K or more groups of threads, and the smallest of the
// groups' maxima has at least K values at or above it.  Some K (ln K + 1) values pass that bar; they are gathered and ranked by
// counting.  Where more pass than the list holds (many equal values), K rounds of a block-wide maximum take over.
#include <float.h>

#include "common.cuh"
#include "host_util.h"
#include "kv_cache.cuh"

namespace bw {
namespace beam {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 64, kMaxBeams = 64;
constexpr int kList = 512;              // candidates that are ranked at once

struct Args {
    int *parent, *token;
    float* score_out;
    unsigned char* ended_out;
    const float* logits;
    long row_stride;
    int vocab;
    const float* score;
    const unsigned char* ended;
    int eos, beams, keep, M, chunks, chunk;
    float2* sums;                       // [M * beams][chunks] maximum, sum of exponentials relative to it
    unsigned long long* best;           // [M * beams][chunks][keep] keys, largest first; 0: none
};

__device__ __forceinline__ uint32_t order32(float f) {
    const uint32_t b = __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order32_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
// Larger value first, then the lower index.
__device__ __forceinline__ unsigned long long key_of(float v, uint32_t index) { return (unsigned long long)order32(v) << 32 | (0xFFFFFFFFu - index); }

struct Cand {
    double score;
    uint32_t at;                        // beam * vocab + token
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.score > b.score || (a.score == b.score && a.at < b.at); }

// Groups of 2^s neighbouring threads, at least `keep` of them: how many threads a group has.
__device__ __forceinline__ int group_size(int keep) {
    int n = kThreads;
    while (kThreads / n < keep) n >>= 1;
    return n;
}

// PER values of a thread in registers.
template <int PER>
__global__ void __launch_bounds__(kThreads) chunk_kernel(const Args a) {
    __shared__ float s_f[kWarps];
    __shared__ float s_max[kWarps];
    __shared__ unsigned long long s_list[kList];
    __shared__ int s_n;
    pdl_trigger();
    pdl_wait();
    const int c = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int v0 = c * a.chunk, n = min(a.vocab - v0, a.chunk);
    const float* x = a.logits + (size_t)row * a.row_stride + v0;
    if (t == 0) s_n = 0;
    float v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = t + kThreads * j;
        v[j] = i < n ? fmaxf(x[i], -INFINITY) : -INFINITY;     // (NaN: -inf)
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = fmaxf(top, v[j]);
    // the bar: the least of the groups' maxima
    const int gs = group_size(a.keep);
    float gm = top;
    for (int o = 1; o < min(gs, 32); o <<= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    float wmax = warp_max(top), wmin = -warp_max(-gm);
    if (lane == 0) { s_max[warp] = wmax; s_f[warp] = wmin; }
    __syncthreads();
    float bmax = s_max[0], bar = INFINITY;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bmax = fmaxf(bmax, s_max[w]);
    if (gs <= 32) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) bar = fminf(bar, s_f[w]);
    } else {
        for (int w = 0; w < kWarps; w += gs / 32) {
            float g = s_max[w];
            for (int e = 1; e < gs / 32; ++e) g = fmaxf(g, s_max[w + e]);
            bar = fminf(bar, g);
        }
    }
    __syncthreads();
    float sum = 0.f;
    if (bmax > -INFINITY) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += __expf(v[j] - bmax);
    }
    sum = warp_sum(sum);
    if (lane == 0) s_f[warp] = sum;
    // what passes the bar
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (v[j] >= bar && v[j] > -INFINITY) {
            const int k = atomicAdd(&s_n, 1);
            if (k < kList) s_list[k] = key_of(v[j], v0 + t + kThreads * j);
        }
    __syncthreads();
    const size_t rec = (size_t)row * a.chunks + c;
    if (t == 0) {
        float all = 0.f;
        for (int w = 0; w < kWarps; ++w) all += s_f[w];
        a.sums[rec] = make_float2(bmax, all);
    }
    unsigned long long* out = a.best + rec * a.keep;
    const int got = s_n;
    if (got <= kList) {
        for (int i = t; i < got; i += kThreads) {
            const unsigned long long k = s_list[i];
            int rank = 0;
            for (int j = 0; j < got; ++j) rank += s_list[j] > k;
            if (rank < a.keep) out[rank] = k;
        }
        for (int i = got + t; i < a.keep; i += kThreads) out[i] = 0;
        return;
    }
    unsigned long long last = ~0ull;
    for (int r = 0; r < a.keep; ++r) {
        unsigned long long k = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const unsigned long long q = key_of(v[j], v0 + t + kThreads * j);
            if (v[j] > -INFINITY && q < last && q > k) k = q;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long q = __shfl_xor_sync(0xffffffffu, k, o);
            k = q > k ? q : k;
        }
        __syncthreads();
        if (lane == 0) s_list[warp] = k;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) k = s_list[w] > k ? s_list[w] : k;
        if (t == 0) out[r] = k;
        last = k;                                              // (0 once there are no more)
    }
}

__global__ void __launch_bounds__(kThreads) merge_kernel(const Args a) {
    __shared__ double s_lse[kMaxBeams];
    __shared__ float s_score[kMaxBeams];
    __shared__ unsigned char s_ended[kMaxBeams];
    __shared__ Cand s_list[kList];
    __shared__ Cand s_w[kWarps];
    __shared__ double s_max[kWarps], s_min[kWarps];
    __shared__ int s_n;
    pdl_trigger();
    pdl_wait();
    const int m = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t == 0) s_n = 0;
    for (int b = warp; b < a.beams; b += kWarps) {
        const float2* rec = a.sums + ((size_t)m * a.beams + b) * a.chunks;
        float mx = -INFINITY;
        for (int c = lane; c < a.chunks; c += 32) mx = fmaxf(mx, rec[c].x);
        mx = warp_max(mx);
        double sum = 0.0;
        for (int c = lane; c < a.chunks; c += 32) {
            const float2 r = rec[c];
            if (r.x > -INFINITY) sum += (double)r.y * exp((double)r.x - (double)mx);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_lse[b] = (double)mx + log(sum);
            s_score[b] = a.score[m * a.beams + b];
            s_ended[b] = a.ended ? a.ended[m * a.beams + b] : 0;
        }
    }
    __syncthreads();
    const int per_beam = a.chunks * a.keep, total = a.beams * per_beam;
    const unsigned long long* best = a.best + (size_t)m * total;
    // Candidate number i; score -inf: none.
    auto cand = [&](int i) {
        const int b = i / per_beam;
        Cand x{-INFINITY, 0xFFFFFFFFu};
        if (s_ended[b]) {
            if (i == b * per_beam && s_score[b] > -INFINITY) x = Cand{(double)s_score[b], (uint32_t)b * a.vocab + a.eos};
            return x;
        }
        const unsigned long long k = best[i];
        if (k == 0) return x;
        const double s = (double)s_score[b] + ((double)order32_value((uint32_t)(k >> 32)) - s_lse[b]);
        if (s > -INFINITY) x = Cand{s, (uint32_t)b * a.vocab + (0xFFFFFFFFu - (uint32_t)k)};
        return x;
    };
    double top = -INFINITY;
    for (int i = t; i < total; i += kThreads) top = fmax(top, cand(i).score);
    const int gs = group_size(a.keep);
    double gm = top, wmax = top;
    for (int o = 1; o < min(gs, 32); o <<= 1) gm = fmax(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    double wmin = gm;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        wmax = fmax(wmax, __shfl_xor_sync(0xffffffffu, wmax, o));
        wmin = fmin(wmin, __shfl_xor_sync(0xffffffffu, wmin, o));
    }
    if (lane == 0) { s_max[warp] = wmax; s_min[warp] = wmin; }
    __syncthreads();
    double bar = INFINITY;
    if (gs <= 32) {
        for (int w = 0; w < kWarps; ++w) bar = fmin(bar, s_min[w]);
    } else {
        for (int w = 0; w < kWarps; w += gs / 32) {
            double g = s_max[w];
            for (int e = 1; e < gs / 32; ++e) g = fmax(g, s_max[w + e]);
            bar = fmin(bar, g);
        }
    }
    for (int i = t; i < total; i += kThreads) {
        const Cand x = cand(i);
        if (x.score >= bar && x.score > -INFINITY) {
            const int k = atomicAdd(&s_n, 1);
            if (k < kList) s_list[k] = x;
        }
    }
    __syncthreads();
    const int got = s_n;
    auto emit = [&](int r, const Cand& x) {
        const size_t o = (size_t)m * a.keep + r;
        const bool some = x.score > -INFINITY;
        const int b = some ? (int)(x.at / (uint32_t)a.vocab) : -1, v = some ? (int)(x.at - (uint32_t)b * a.vocab) : -1;
        a.parent[o] = b;
        a.token[o] = v;
        a.score_out[o] = (float)x.score;
        if (a.ended_out) a.ended_out[o] = some && (s_ended[b] || v == a.eos);
    };
    if (got <= kList) {
        for (int i = t; i < got; i += kThreads) {
            const Cand x = s_list[i];
            int rank = 0;
            for (int j = 0; j < got; ++j) rank += before(s_list[j], x);
            if (rank < a.keep) emit(rank, x);
        }
        for (int i = got + t; i < a.keep; i += kThreads) emit(i, Cand{-INFINITY, 0xFFFFFFFFu});
        return;
    }
    Cand last{INFINITY, 0};
    for (int r = 0; r < a.keep; ++r) {
        Cand x{-INFINITY, 0xFFFFFFFFu};
        for (int i = t; i < total; i += kThreads) {
            const Cand y = cand(i);
            if ((r == 0 || before(last, y)) && before(y, x)) x = y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand y{__shfl_xor_sync(0xffffffffu, x.score, o), __shfl_xor_sync(0xffffffffu, x.at, o)};
            if (before(y, x)) x = y;
        }
        __syncthreads();
        if (lane == 0) s_w[warp] = x;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w)
            if (before(s_w[w], x)) x = s_w[w];
        if (t == 0) emit(r, x);
        last = x;
    }
}

// Values of a chunk: 2,048 (eight a thread) where that leaves a few blocks per SM at most, else 8,192.
static int chunk_of(int vocab, long rows) {
    return rows * ((vocab + 2047) / 2048) <= 8L * sm_count(current_device()) ? 2048 : 8192;
}
static size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t bytes_of(long rows, int chunks, int keep) {
    return round16((size_t)rows * chunks * sizeof(float2)) + (size_t)rows * chunks * keep * sizeof(unsigned long long);
}
static bool sizes_ok(int vocab, int beams, int keep, int M) {
    return vocab >= 1 && beams >= 1 && beams <= kMaxBeams && keep >= 1 && keep <= kMaxKeep && M >= 1 && (long)M * beams <= 65535 &&
           (long)beams * vocab < 0x7FFFFFFFL;
}

}  // namespace beam
}  // namespace bw

using namespace bw;

extern "C" size_t bw_beam_select_scratch_bytes(int vocab, int beams, int keep, int M) {
    if (!beam::sizes_ok(vocab, beams, keep, M)) return 0;
    return beam::bytes_of((long)M * beams, (vocab + 2047) / 2048, keep);
}

extern "C" int bw_beam_select(int* parent_out, int* token_out, float* score_out, unsigned char* ended_out_or_null, const float* logits,
                              long row_stride, int vocab, const float* score, const unsigned char* ended_or_null, int eos_id, int beams, int keep,
                              int M, void* scratch, size_t scratch_bytes, void* stream) {
    if (!beam::sizes_ok(vocab, beams, keep, M) || !parent_out || !token_out || !score_out || !logits || !score || !scratch) return cudaErrorInvalidValue;
    if (row_stride < vocab || (ended_or_null && (eos_id < 0 || eos_id >= vocab)) || !kv::aligned(scratch, 16)) return cudaErrorInvalidValue;
    const long rows = (long)M * beams;
    beam::Args a{};
    a.chunk = beam::chunk_of(vocab, rows);
    a.chunks = (vocab + a.chunk - 1) / a.chunk;
    if (scratch_bytes < beam::bytes_of(rows, a.chunks, keep)) return cudaErrorInvalidValue;
    a.parent = parent_out; a.token = token_out; a.score_out = score_out; a.ended_out = ended_out_or_null;
    a.logits = logits; a.row_stride = row_stride; a.vocab = vocab; a.score = score; a.ended = ended_or_null;
    a.eos = eos_id; a.beams = beams; a.keep = keep; a.M = M;
    a.sums = static_cast<float2*>(scratch);
    a.best = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(scratch) + beam::round16((size_t)rows * a.chunks * sizeof(float2)));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)a.chunks, (unsigned)rows);
    cudaError_t e = a.chunk == 2048 ? launch_pdl(beam::chunk_kernel<8>, grid, dim3(beam::kThreads), 0, st, a)
                                    : launch_pdl(beam::chunk_kernel<32>, grid, dim3(beam::kThreads), 0, st, a);
    if (e == cudaSuccess) e = launch_pdl(beam::merge_kernel, dim3((unsigned)M), dim3(beam::kThreads), 0, st, a);
    count_launch(2);
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
