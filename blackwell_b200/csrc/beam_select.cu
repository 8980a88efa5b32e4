// Beam search's selection: of the candidates  score[b] + log_softmax(logits[b])[v]  of a request's beams the best few.
//
// Two launches, or one of clusters that joins them.  The first reads the logits once, a stretch of a row per block, 4,096 values at a time with the next ones in flight.  A
// warp works by itself: running maxima and sums of exponentials per lane, and a list of the values that may be among the `keep` largest of
// the stretch (within a row the order of the candidates is that of the logits).  What enters the list is at or above a bar: the
// smallest of the running maxima of `keep` or more groups of the block's threads.  At least `keep` values lie there, of the first n some keep *
// (ln keep + 1), so that after the first turns hardly a warp has one.  The maxima only grow, so that warps share them without waiting for
// each other: a stale one lowers the bar.  A list that has grown is cut to its best.  The second launch, a block per request, forms the rows' log-sums and ranks the
// stretches' candidates across the beams, scores in 64 bits: two beams' candidates may lie closer to each other than 32 bits tell apart.
// The exponentials and their sums are 32-bit, taken of differences that are exact where they matter; a log-sum is right to some 1e-7.
// Measured (16 x 8 beams of 151,643 tokens, 78 MB): 24.4 us, 3.2 TB/s, of which the merge and its launch are 4; the first launch alone is bound
// by the instructions that a value takes, not by memory (the exponentials some 5 us of it).  One request of 8 or 16 such beams, whose 2,432 or 8,192
// candidates do not fit shared memory: 12.6 and 20.4 us.
#include <float.h>

#include <mutex>

#include "common.cuh"
#include "host_util.h"
#include "kv_cache.cuh"
#include "lm_device.cuh"

namespace bw {
namespace beam {

using lm::exp2_fast;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 64, kMaxBeams = 64;
constexpr int kVec = 4;                       // 16-byte vectors of a thread in flight
constexpr int kTurn = kThreads * kVec;        // vectors a block takes at once
constexpr int kGrown = 128;                   // entries from which a warp's list is cut to the best
constexpr int kList = kGrown + 32 * 4 * kVec; // ... and one turn that enters whole
constexpr int kStaged = 2048;                 // candidates of a request that the merge holds in shared memory
constexpr int kMaxLists = 64 * kWarps;        // stretches of a request's beams, at most: two per lane of the merge's warps

struct Args {
    int *parent, *token;
    float* score_out;
    unsigned char* ended_out;
    const float* logits;
    long row_stride;
    int vocab;
    const float* score;
    const unsigned char* ended;
    int eos, beams, keep, M, chunks, chunk;     // stretches of a row, their length in vectors
    float2* sums;                       // [M * beams][chunks] maximum, sum of exponentials relative to it
    unsigned long long* best;           // [M * beams][chunks][keep] keys, largest first; 0: none
};

__device__ __forceinline__ uint32_t order32(float f) {
    const uint32_t b = __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order32_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
// Larger value first, then the lower index; the zeros are one value.
__device__ __forceinline__ unsigned long long key_of(float v, uint32_t index) { return (unsigned long long)order32(v + 0.f) << 32 | (0xFFFFFFFFu - index); }

// A candidate of the merge: its score as an integer that orders as the score does (64-bit comparisons of floats have a long latency; ranking
// is a chain of them), 0: none.
struct Cand {
    unsigned long long score;
    uint32_t at;                        // beam * vocab + token
};
__device__ __forceinline__ unsigned long long order64(double d) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(d + 0.0);   // (-0 becomes +0)
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double order64_value(unsigned long long k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k)); }

__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xffffffffu, k, o);
        k = q > k ? q : k;
    }
    return k;
}
// The best `keep` of the warp's n keys to the front of its list, largest first; zeros where there are fewer.
__device__ __forceinline__ void cut_list(unsigned long long* list, int n, int keep, int lane) {
    unsigned long long last = ~0ull, mine[2] = {0, 0};
    __syncwarp();
    for (int r = 0; r < keep; ++r) {
        unsigned long long k = 0;
        for (int i = lane; i < n; i += 32) {
            const unsigned long long q = list[i];
            if (q < last && q > k) k = q;
        }
        last = warp_max_key(k);
        if ((r & 31) == lane) mine[r >> 5] = last;
        if (last == 0) break;
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 32 * e < keep) list[lane + 32 * e] = mine[e];
    __syncwarp();
}

// Sum of exp(v - to) over a thread's values, two at a time.
__device__ __forceinline__ float exponentials(const float4 (&v)[kVec], float to) {
    unsigned long long part[2];
    const unsigned long long minus = pair_of(-to, -to), scale = pair_of(kLog2e, kLog2e);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            unsigned long long d;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(e ? pair_of(v[j].z, v[j].w) : pair_of(v[j].x, v[j].y)), "l"(minus));
            asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(scale));
            float lo, hi;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d));
            const unsigned long long x = pair_of(exp2_fast(lo), exp2_fast(hi));
            if (j == 0) part[e] = x;
            else asm("add.rn.f32x2 %0, %0, %1;" : "+l"(part[e]) : "l"(x));
        }
    float p[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) asm("mov.b64 {%0, %1}, %2;" : "=f"(p[2 * e]), "=f"(p[2 * e + 1]) : "l"(part[e]));
    return (p[0] + p[1]) + (p[2] + p[3]);
}

// Which of several candidates of the same score comes first: the lower beam, within a beam the larger logit, as inside a list (two logits may differ by
// less than their 64-bit scores show), then the lower token.  x: the lane's two, of which `in` (by bits) are among them; bit 2: the winner is this
// lane's, of number bit 0.  rows: the request's logits.  (A call: hardly ever needed, and the rounds are short.)
__device__ __noinline__ int first_of_equal(uint32_t at0, uint32_t at1, int in, const float* rows, long row_stride, uint32_t vocab) {
    auto logit = [&](uint32_t at) {
        const uint32_t b = at / vocab;
        return order32(rows[(size_t)b * row_stride + (at - b * vocab)] + 0.f);
    };
    const uint32_t beam0 = in & 1 ? at0 / vocab : 0xFFFFFFFFu, beam1 = in & 2 ? at1 / vocab : 0xFFFFFFFFu;
    const uint32_t beam = __reduce_min_sync(0xffffffffu, min(beam0, beam1));
    const uint32_t v0 = beam0 == beam ? logit(at0) : 0, v1 = beam1 == beam ? logit(at1) : 0;     // (an ended beam's one may have any bits)
    const uint32_t v = __reduce_max_sync(0xffffffffu, max(v0, v1));
    const uint32_t c0 = beam0 == beam && v0 == v ? at0 : 0xFFFFFFFFu, c1 = beam1 == beam && v1 == v ? at1 : 0xFFFFFFFFu;
    const uint32_t at = __reduce_min_sync(0xffffffffu, min(c0, c1));
    return c0 == at ? 4 : c1 == at ? 5 : 0;
}
// The best of up to 64 sorted lists, two per lane, one after the other: head(l, i) is entry i of list l (score 0: none), emit(r, cand)
// takes the r-th best, by the lane that holds it.  A round is three warp-wide integer reductions; only the winner's list moves on.
template <typename Head, typename Emit>
__device__ __forceinline__ void tournament(int lists, int keep, int lane, const float* rows, long row_stride, uint32_t vocab, const Head& head, const Emit& emit) {
    Cand x[2];
    int i[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e) x[e] = lane + 32 * e < lists ? head(lane + 32 * e, 0) : Cand{0, 0};
    for (int r = 0; r < keep; ++r) {
        int e = x[1].score > x[0].score;
        const unsigned long long y = e ? x[1].score : x[0].score;
        const uint32_t hi = (uint32_t)(y >> 32), lo = (uint32_t)y;
        const uint32_t mhi = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t mlo = __reduce_max_sync(0xffffffffu, hi == mhi ? lo : 0u);
        bool best = hi == mhi && lo == mlo;
        const bool both = x[0].score == x[1].score;
        if (mhi == 0 && mlo == 0) {
            if (lane == 0)
                for (; r < keep; ++r) emit(r, Cand{0, 0});
            break;
        }
        if (__reduce_add_sync(0xffffffffu, best ? both ? 2u : 1u : 0u) > 1) {
            const int w = first_of_equal(x[0].at, x[1].at, !best ? 0 : both ? 3 : 1 << e, rows, row_stride, vocab);
            best = w != 0;
            e = w & 1;
        }
        if (best) {
            emit(r, e ? x[1] : x[0]);
            if (e) x[1] = ++i[1] < keep ? head(lane + 32, i[1]) : Cand{0, 0};
            else x[0] = ++i[0] < keep ? head(lane, i[0]) : Cand{0, 0};
        }
    }
    __syncwarp();
}

// The rest of request m: log-sums, then the best of the stretches' candidates, whose scores are formed before, all at once: a round that forms the
// winner's next one takes 1,000 cycles, one that finds it 300.  s_key, s_at: kStaged each.  kFew: 64 lists at most.
template <bool kFew>
__device__ __forceinline__ void merge(const Args& a, int m, unsigned long long* s_key, uint32_t* s_at) {
    __shared__ double s_lse[kMaxBeams];
    __shared__ float s_score[kMaxBeams];
    __shared__ unsigned char s_ended[kMaxBeams];
    __shared__ Cand s_best[kFew ? 1 : kWarps][kMaxKeep], s_out[kMaxKeep];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lists = a.beams * a.chunks, total = lists * a.keep;
    const unsigned long long* best = a.best + (size_t)m * total;
    const bool staged = total <= kStaged;
    if (staged)
        for (int i = t; i < total; i += kThreads) s_key[i] = best[i];
    for (int b = warp; b < a.beams; b += kWarps) {
        const float2* rec = a.sums + ((size_t)m * a.beams + b) * a.chunks;
        const float2 one = lane < a.chunks ? rec[lane] : make_float2(-INFINITY, 0.f);
        float mx = one.x;
        for (int c = lane + 32; c < a.chunks; c += 32) mx = fmaxf(mx, rec[c].x);
        mx = warp_max(mx);
        float sum = one.x > -INFINITY ? one.y * exp2f((one.x - mx) * kLog2e) : 0.f;
        for (int c = lane + 32; c < a.chunks; c += 32) {
            const float2 r = rec[c];
            if (r.x > -INFINITY) sum += r.y * exp2f((r.x - mx) * kLog2e);
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            // log sum = k ln 2 + log of what is left, which lies in [1, 2): its 32-bit rounding is under 2^-24
            int k = 0;
            float left = sum;
            if (sum >= 1.f && sum < INFINITY) {
                k = (int)(__float_as_uint(sum) >> 23) - 127;
                left = __uint_as_float((__float_as_uint(sum) & 0x7FFFFFu) | 0x3F800000u);
            }
            s_lse[b] = (double)mx + fma((double)k, 0.6931471805599453, (double)logf(left));
            s_score[b] = a.score[m * a.beams + b];
            s_ended[b] = a.ended ? a.ended[m * a.beams + b] : 0;
        }
    }
    __syncthreads();
    // Entry i of list l (a beam's stretch); an ended beam has one, its first stretch's.
    auto formed = [&](int l, int i, unsigned long long k) {
        const int b = l / (uint32_t)a.chunks;
        Cand x{0, 0};
        if (s_ended[b]) {
            if (l == b * a.chunks && i == 0 && s_score[b] > -INFINITY) x = Cand{order64((double)s_score[b]), (uint32_t)b * a.vocab + a.eos};
            return x;
        }
        if (k == 0) return x;
        const double s = (double)s_score[b] + ((double)order32_value((uint32_t)(k >> 32)) - s_lse[b]);
        if (s > -INFINITY) x = Cand{order64(s), (uint32_t)b * a.vocab + (0xFFFFFFFFu - (uint32_t)k)};
        return x;
    };
    if (staged) {
        for (int j = t; j < total; j += kThreads) {
            const int l = j / (uint32_t)a.keep;
            const Cand x = formed(l, j - l * a.keep, s_key[j]);
            s_key[j] = x.score;
            s_at[j] = x.at;
        }
        __syncthreads();
    }
    auto head = [&](int l, int i) {
        const int j = l * a.keep + i;
        return staged ? Cand{s_key[j], s_at[j]} : formed(l, i, best[(size_t)j]);
    };
    auto out = [&](int r, const Cand& x) { s_out[r] = x; };
    const uint32_t vocab = a.vocab;
    const float* rows = a.logits + (size_t)m * a.beams * a.row_stride;
    if (kFew || lists <= 64) {
        if (warp != 0) return;
        tournament(lists, a.keep, lane, rows, a.row_stride, vocab, head, out);
    } else {
        const int per = (lists + kWarps - 1) / kWarps, l0 = min(warp * per, lists);
        tournament(min(per, lists - l0), a.keep, lane, rows, a.row_stride, vocab, [&](int l, int i) { return head(l0 + l, i); }, [&](int r, const Cand& x) { s_best[kFew ? 0 : warp][r] = x; });
        __syncthreads();
        if (warp != 0) return;
        tournament(kWarps, a.keep, lane, rows, a.row_stride, vocab, [&](int l, int i) { return s_best[kFew ? 0 : l][i]; }, out);
    }
    for (int r = lane; r < a.keep; r += 32) {            // (the tournament ends with its warp's writes in place)
        const Cand x = s_out[r];
        const size_t o = (size_t)m * a.keep + r;
        const bool some = x.score != 0;
        const int b = some ? (int)(x.at / vocab) : -1, v = some ? (int)(x.at - (uint32_t)b * vocab) : -1;
        a.parent[o] = b;
        a.token[o] = v;
        a.score_out[o] = some ? (float)order64_value(x.score) : -INFINITY;
        if (a.ended_out) a.ended_out[o] = some && (s_ended[b] || v == a.eos);
    }
}

__global__ void __launch_bounds__(kThreads) merge_kernel(const Args a) {
    __shared__ unsigned long long s_key[kStaged];
    __shared__ uint32_t s_at[kStaged];
    pdl_trigger();
    pdl_wait();
    merge<false>(a, blockIdx.x, s_key, s_at);
}

// kFused: a request's blocks are a cluster, whose first goes on with the merge.
template <bool kFused>
__global__ void __launch_bounds__(kThreads, 4) chunk_kernel(const Args a) {
    __shared__ unsigned long long s_list[kWarps][kList], s_all[kWarps * kMaxKeep];
    __shared__ float s_f[kWarps], s_g[kWarps];
    __shared__ uint32_t s_group[64];
    __shared__ int s_n[kWarps];
    const int c = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const float* x = a.logits + (size_t)row * a.row_stride;
    const int skew = (int)(reinterpret_cast<uintptr_t>(x) >> 2 & 3);     // vector q: elements 4 q - skew ...
    const int q0 = c * a.chunk, q1 = min(q0 + a.chunk, (a.vocab + skew + 3) / 4);
    pdl_trigger();
    pdl_wait();
    auto load = [&](int base, float4 (&v)[kVec]) {
        if (4 * base >= skew && 4 * (base + kTurn) - skew <= a.vocab && base + kTurn <= q1) {
            const float4* p = reinterpret_cast<const float4*>(x - skew) + base + t;
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] = p[kThreads * j];
            return;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) {                                 // a row's ends
            const int q = base + kThreads * j + t, i = 4 * q - skew;
            float e[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) e[d] = q < q1 && i + d >= 0 && i + d < a.vocab ? x[i + d] : -INFINITY;
            v[j] = make_float4(e[0], e[1], e[2], e[3]);
        }
    };
    float4 next[kVec];
    load(q0, next);
    if (t < 64) s_group[t] = 0;                                          // (below every value)
    __syncthreads();
    unsigned long long* list = s_list[warp];
    float m[2] = {-INFINITY, -INFINITY}, sum = 0.f, ground = -FLT_MAX;     // maxima of the lane's even and odd vectors
    int n = 0, groups = 1;
    while (groups < a.keep) groups <<= 1;
    auto bar_of = [&]() {                                                // the smallest of the groups' maxima so far
        const volatile uint32_t* g = s_group;
        uint32_t low = lane < groups ? g[lane] : 0xFFFFFFFFu;
        if (groups > 32) low = min(low, g[32 + lane]);
        return order32_value(__reduce_min_sync(0xffffffffu, low));
    };
    for (int base = q0; base < q1; base += kTurn) {
        float4 v[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = next[j];
        if (base + kTurn < q1) load(base + kTurn, next);
        const float old = fmaxf(m[0], m[1]);
        float top[2] = {-INFINITY, -INFINITY};                           // (a NaN is no maximum)
#pragma unroll
        for (int j = 0; j < kVec; ++j) top[j & 1] = fmaxf(top[j & 1], fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
        m[0] = fmaxf(m[0], top[0]);
        m[1] = fmaxf(m[1], top[1]);
        const float to = fmaxf(m[0], m[1]), best = fmaxf(top[0], top[1]);
        if (to > -INFINITY) {
            const float kept = sum * exp2_fast((old - to) * kLog2e);
            sum = kept + exponentials(v, to);
            if (sum != sum) {                                            // a NaN counts as -inf (and +inf leaves NaN here)
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    v[j] = make_float4(fmaxf(v[j].x, -INFINITY), fmaxf(v[j].y, -INFINITY), fmaxf(v[j].z, -INFINITY), fmaxf(v[j].w, -INFINITY));
                sum = kept + exponentials(v, to);
            }
        }
        // group (thread mod G), or with G = 64 (lane) and (32 + lane) of the lanes' two maxima
        if (groups > 32) {
            atomicMax(&s_group[lane], order32(m[0]));
            atomicMax(&s_group[32 + lane], order32(m[1]));
        } else {
            float g = to;
            for (int o = 16; o >= groups; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
            if (lane < groups) atomicMax(&s_group[lane], order32(g));
        }
        if (base == q0) __syncthreads();                                 // the first bar is that of the block's values, not of a warp's
        else __syncwarp();
        const float bar = bar_of();
        if (__any_sync(0xffffffffu, best >= fmaxf(bar, ground))) {
            const uint32_t i0 = (uint32_t)(4 * (base + t) - skew);
            const float least = fmaxf(bar, ground);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t who = __ballot_sync(0xffffffffu, e[d] >= least);
                    if (who) {                                           // (hardly ever: a branch costs less than what it skips)
                        if (e[d] >= least) list[n + __popc(who & ((1u << lane) - 1))] = key_of(e[d], i0 + 4 * kThreads * j + d);
                        n += __popc(who);
                    }
                }
            }
            if (n > kGrown) {
                cut_list(list, n, a.keep, lane);
                ground = order32_value((uint32_t)(list[a.keep - 1] >> 32) + 1);   // the next float: what equals the last one comes too late
                n = a.keep;
                __syncwarp();
            }
        }
    }
    // the block's maximum and sum, and the best of the warps' lists
    const float mine = fmaxf(m[0], m[1]), wm = warp_max(mine);
    if (lane == 0) s_g[warp] = wm;
    __syncthreads();
    {                                                                    // what is at or above the last bar
        const float bar = fmaxf(bar_of(), -FLT_MAX);
        int left = 0;
        for (int i0 = 0; i0 < n; i0 += 32) {
            const unsigned long long k = i0 + lane < n ? list[i0 + lane] : 0;
            const bool in = k != 0 && order32_value((uint32_t)(k >> 32)) >= bar;
            const uint32_t who = __ballot_sync(0xffffffffu, in);         // (all have read before any writes, at or before where it read)
            if (in) list[left + __popc(who & ((1u << lane) - 1))] = k;
            left += __popc(who);
            __syncwarp();
        }
        n = left;
    }
    if (lane == 0) s_n[warp] = n;
    if (__syncthreads_or(n > kMaxKeep)) {
        if (n > a.keep) cut_list(list, n, a.keep, lane);
        n = min(n, a.keep);
        if (lane == 0) s_n[warp] = n;
        __syncthreads();
    }
    float top = s_g[0];
    int all = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        top = fmaxf(top, s_g[w]);
        at = w == warp ? all : at;
        all += s_n[w];
    }
    sum = warp_sum(mine > -INFINITY ? sum * exp2_fast((mine - top) * kLog2e) : 0.f);
    if (lane == 0) s_f[warp] = sum;
    for (int i = lane; i < n; i += 32) s_all[at + i] = list[i];
    __syncthreads();
    const size_t rec = (size_t)row * a.chunks + c;
    unsigned long long* out = a.best + rec * a.keep;
    for (int i = t; i < all; i += kThreads) {
        const unsigned long long k = s_all[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < all; ++j) rank += s_all[j] > k;
        if (rank < a.keep) out[rank] = k;
    }
    if (t >= all && t < a.keep) out[t] = 0;
    if (t == 0) {
        float whole = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) whole += s_f[w];
        a.sums[rec] = make_float2(top, whole);
    }
    if (kFused) {
        cluster_sync_all();
        const int m = row / (uint32_t)a.beams;
        static_assert(kWarps * kList * 8 >= kStaged * 12, "the merge's candidates lie over the lists");
        if (c == 0 && row == m * a.beams) merge<true>(a, m, s_list[0], reinterpret_cast<uint32_t*>(s_list[0] + kStaged));
    }
}

// Stretches of a row: whole turns, four blocks per SM where that many are to be had.  A few requests that a cluster each reads in three turns or fewer:
// one launch.  On the device both take much the same (1 x 4 beams of 32,768 tokens 7.2 us, in two launches 6.4), but a launch costs the caller 2 us:
// calls in a row took 9 instead of 11.  skew: elements that rows may start behind a 16-byte boundary.
constexpr int kFusedBlocks = 16, kFusedTurns = 3;
static bool stretches(int vocab, int skew, int beams, long rows, int sms, Args* a) {
    const int vectors = (vocab + skew + 3) / 4, turns = (vectors + kTurn - 1) / kTurn;
    int most = kFusedBlocks / beams;
    most = most > turns ? turns : most;
    const bool fused = most > 0 && rows * most <= 2L * sms && (turns + most - 1) / most <= kFusedTurns;
    long n = fused ? most : 4L * sms / rows;
    n = n > kMaxLists / beams ? kMaxLists / beams : n;
    n = n < 1 ? 1 : n > turns ? turns : n;
    a->chunk = (int)((turns + n - 1) / n) * kTurn;
    a->chunks = (vectors + a->chunk - 1) / a->chunk;
    return fused;
}
static size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t bytes_of(long records, int keep) {
    return round16((size_t)records * sizeof(float2)) + (size_t)records * keep * sizeof(unsigned long long);
}
static bool sizes_ok(int vocab, int beams, int keep, int M) {
    return vocab >= 1 && beams >= 1 && beams <= kMaxBeams && keep >= 1 && keep <= kMaxKeep && M >= 1 && (long)M * beams <= 65535 &&
           (long)beams * vocab <= 0x7FFF0000L;   // (vectors of a turn past the end are counted in 32 bits)
}

}  // namespace beam
}  // namespace bw

using namespace bw;

extern "C" size_t bw_beam_select_scratch_bytes(int vocab, int beams, int keep, int M) {
    if (!beam::sizes_ok(vocab, beams, keep, M)) return 0;
    const long rows = (long)M * beams, most = 4L * sm_count(current_device());   // (records of any smaller call too)
    return beam::bytes_of(rows > most ? rows : most, keep);
}

extern "C" int bw_beam_select(int* parent_out, int* token_out, float* score_out, unsigned char* ended_out_or_null, const float* logits,
                              long row_stride, int vocab, const float* score, const unsigned char* ended_or_null, int eos_id, int beams, int keep,
                              int M, void* scratch, size_t scratch_bytes, void* stream) {
    if (!beam::sizes_ok(vocab, beams, keep, M) || !parent_out || !token_out || !score_out || !logits || !score || !scratch) return cudaErrorInvalidValue;
    if (row_stride < vocab || (ended_or_null && (eos_id < 0 || eos_id >= vocab)) || !kv::aligned(scratch, 16)) return cudaErrorInvalidValue;
    if (keep != beams && (score_out == score || (ended_or_null && ended_out_or_null == ended_or_null))) return cudaErrorInvalidValue;   // (other requests' are still read)
    const long rows = (long)M * beams;
    beam::Args a{};
    const int skew = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && row_stride % 4 == 0 ? 0 : 3;
    const bool fused = beam::stretches(vocab, skew, beams, rows, sm_count(current_device()), &a);
    if (scratch_bytes < beam::bytes_of(rows * a.chunks, keep)) return cudaErrorInvalidValue;
    a.parent = parent_out; a.token = token_out; a.score_out = score_out; a.ended_out = ended_out_or_null;
    a.logits = logits; a.row_stride = row_stride; a.vocab = vocab; a.score = score; a.ended = ended_or_null;
    a.eos = eos_id; a.beams = beams; a.keep = keep; a.M = M;
    a.sums = static_cast<float2*>(scratch);
    a.best = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(scratch) + beam::round16((size_t)rows * a.chunks * sizeof(float2)));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)a.chunks, (unsigned)rows);
    if (fused) {
        static std::once_flag once[kMaxDevices];
        std::call_once(once[current_device()], [] { cudaFuncSetAttribute(beam::chunk_kernel<true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(beam::kThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = grid.x;
        attr[1].val.clusterDim.y = beams;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, beam::chunk_kernel<true>, a);
        count_launch(1);
        return e != cudaSuccess ? e : cudaPeekAtLastError();
    }
    cudaError_t e = launch_pdl(beam::chunk_kernel<false>, grid, dim3(beam::kThreads), 0, st, a);
    if (e == cudaSuccess) e = launch_pdl(beam::merge_kernel, dim3((unsigned)M), dim3(beam::kThreads), 0, st, a);
    count_launch(2);
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
