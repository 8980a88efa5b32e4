// Attention of a few rows per sequence (one token, or the nodes of a drafted tree) over a cached context, on the warp-level tensor
// cores (mma.sync m16n8k16, f16 x f16 -> f32).
//
//   o_r = sum_t softmax_t(q_r k_t / sqrt(128)) v_t     over the rows t that r sees
//
// A query row r is a node and one of the query heads that share the kv head (r = node * group + head).  The products are formed
// transposed, with the cache as the 16-row operand and eight query rows as the columns, so that few rows waste little:
//   S^T [16 positions x 8 rows] = K Q^T,   O^T [16 dimensions x 8 rows] = V^T P^T
// A warp takes 16 positions at a time for all 8 * NT rows of its block; its softmax state and the unnormalised O^T stay in registers.
// P goes from the accumulator layout to the operand layout by movmatrix.  e4m3 codes become f16 exactly (no rounding); the key scale
// multiplies the score, the value scale the probability.  What the f16 operand has to hold is that product: a row's reference is the maximum of
// score + log2(value scale) over what it sees, for its sum as well, so that neither a row that it does not see nor one that it hardly weighs takes
// bits from it.  Scales are taken relative to the size of the warp's first (a power of two), so that scores and references are of one size.
// fp32 activations: Q and P are split in an f16 high part and an f16 remainder (22 significant bits) and multiplied twice, or, with four
// rows or fewer (kPair), once with the remainders in the other four columns; bfloat16 activations: once, which rounds P to 11 bits where
// the result keeps 8.  Each query row is brought to a maximum of 1 to 2 by a power
// of two first.
// The running maximum moves only when a score exceeds the reference by more than 2^14 / 2^6: otherwise no lane needs another's score.  The
// tensor core's sums are cut at 24 bits: with fp32 activations a tile's P V starts at zero and is added to O by a rounded addition.
// Measured (32 / 8 heads, fp32, 8 bits): 32 sequences of 4,096 to 8,192 positions 75 us, 5.6 TB/s; 8 of 2,000 to 4,000 15 us; one of 2,048 6.7 us, most
// of it the chain of a launch, the position, the first tile from memory and the merge inside the cluster.  What it took: the scales with the tiles by
// cp.async (loaded to registers a tile ahead: 92 us), queries brought to their place once per block (by every warp: + 2,000 cycles), and the remainders in
// the idle columns (8 us at 32 sequences).  Trees of 17 to 32 rows a head have two warps per scheduler (255 registers).  32 of 8 nodes over 2,000 to 4,000
// positions, 8 bits: 119 us in fp32, 83 in bf16, the tensor pipe at 38 % and issue at 36: the waits between dependent instructions, then mma.sync itself.  4 of
// 8 nodes over 1,000 positions, 28 / 4 heads, binary16: 13.9 us, tensor pipe 9 %, issue 20 %: start, barriers and the chain of two tiles a warp.  Tried and not kept: an equal stretch of all contexts per block with records
// and a merge (10 us more below 16,000 positions, as much beyond).
#pragma once
#include <float.h>

#include "attention_mma.cuh"
#include "common.cuh"
#include "kv_cache.cuh"
#include "lm_device.cuh"

namespace bw {
namespace tree {

using kv::kHd;
constexpr int kMaxNodes = 64;
constexpr int kTile = 16;               // positions a warp takes at once
constexpr int kPart = kHd + 4;          // floats of a partial record: outputs, maximum, sum, padding
constexpr float kHead = 6.f, kSlack = 14.f;   // P up to 2^6 when the maximum is new, 2^14 before it is moved
constexpr float kLeastScale = -90.f;    // log2; a smaller value scale counts as this one in the reference: sums of P without it stay below 2^104 a position

struct Args {
    void* out;                          // [M * T][nq * 128]
    const void* q;                      // the same
    kv::View c;
    const int *first, *count;
    const unsigned long long* mask;     // [M * T] or NULL: node j <= i
    int nq, M, T, group, rows, tiles;   // rows = T * group query rows per kv head, in `tiles` blocks of 8 * NT
    int nsplit, cluster;                // blocks that share a context; those that join as a cluster
    float* part;                        // [M][heads][rows][nsplit / cluster][kPart] where there are several; tcgen05 kernel: [2 * blocks][kPart / 4][rec_rows][4]
    // tcgen05 kernel
    int flat, blocks, pairs, groups, group_rows, rec_rows;   // work in a line; heads and row groups of 128 or 256 rows in all
    int* cum;                           // tiles before each sequence; from kPlanned on, [blocks + 1], where each block's stretch starts
    float* kept;                        // fp32: [blocks][2][32][128][4]
    int* status;
};

template <int NT, bool kCoded>
struct Shape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kStages = NT > 2 && !kCoded ? 2 : 3;              // (two blocks fit an SM)
    static constexpr int kWarps = NT == 1 && kCoded ? 8 : 4;               // two blocks per SM, as many warps as the registers allow
    static constexpr int kSide = kTile * kHd * (kCoded ? 1 : 2);           // bytes of 16 K or V rows
    static constexpr int kStage = 2 * kSide + (kCoded ? 2 * kTile * 4 : 0);  // ... and their scales
    static constexpr int kRing = kStages * kStage;
    static constexpr int kO = kRows * kHd * 4;                             // a warp's O, over its stages once they have drained
    static constexpr int kPerWarp = kRing > kO ? kRing : kO;
    static constexpr int kQ = 8 * NT * 32 * 16;                            // the query operand, [k-step][tile][lane] high parts and remainders
    static constexpr int kSmem = kWarps * kPerWarp + kQ;
};

// f16 pairs of two e4m3 codes each (exact): the low and the high half of a word.
__device__ __forceinline__ void codes_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with a sum that starts at zero.
__device__ __forceinline__ void mma_f16_new(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 4 bytes to shared memory on their way, zeros without `in`.
__device__ __forceinline__ void cp_async4z(uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
// (x, y) += (a, b), as one instruction.
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 v, f;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 f, {%2, %3};\n\tadd.rn.f32x2 v, v, f;\n\tmov.b64 {%0, %1}, v;\n\t}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ float4 ld_dsmem4(uint32_t addr, uint32_t rank) {
    uint32_t ra;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ra) : "memory");
    return v;
}
// Power of two at or below |x| (1 for zero and what has no such), and its reciprocal.
__device__ __forceinline__ float2 binade(float x) {
    uint32_t e = __float_as_uint(x) >> 23 & 255;
    e = e < 1 ? 127 : min(max(e, 2u), 252u);
    return make_float2(__uint_as_float(e << 23), __uint_as_float((254 - e) << 23));
}

// The power of two that value scales are taken relative to, at or above their largest (bits of its magnitude).
__device__ __forceinline__ float scale_unit(uint32_t top) { return __uint_as_float(min(max((top + 0x7FFFFFu) & 0x7F800000u, 87u << 23), 167u << 23)); }
__device__ __forceinline__ float scale_log2(float relative) { return fmaxf(__log2f(fabsf(relative)), kLeastScale); }

// 2^(from - to), to >= from, in two factors: references that value scales keep far apart (or rows of scale zero) may differ by more than the 2^126 of
// one, and a sum of probabilities, which is as far from 1, has to outlast that.  Sums of P V that far below do not count.
template <bool kFar>
__device__ __forceinline__ float2 step(float from, float to) {
    const float h = lm::exp2_fast(kFar ? 0.5f * (from - to) : from - to);
    return make_float2(h, kFar ? h : 1.f);
}

// What a sequence's rows see: positions [0, first) all of them, node j (position first + j) by bit j of a row's mask.
__device__ __forceinline__ unsigned long long low_bits(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ int node_count(const Args& a, int m) { return a.count ? max(0, min(a.count[m], a.T)) : a.T; }
__device__ __forceinline__ unsigned long long mask_of(const Args& a, int m, int node, int nodes) {
    return (a.mask ? a.mask[(size_t)m * a.T + node] : low_bits(node + 1)) & low_bits(nodes);
}

template <int NT, bool kCoded, typename A, bool kPair>
__global__ void __launch_bounds__(Shape<NT, kCoded>::kWarps * 32, 2) attend_kernel(const Args a) {
    using Sh = Shape<NT, kCoded>;
    constexpr int kWarps = Sh::kWarps;
    constexpr bool kSplit = sizeof(A) == 4 && !kPair;   // fp32 activations: two products
    constexpr int kRowOf = kPair ? 3 : 7;               // row of a column, in bits
    static_assert(!kPair || (NT == 1 && sizeof(A) == 4), "four rows");
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ unsigned long long s_mask[Sh::kRows];
    __shared__ float s_m[kWarps][Sh::kRows], s_l[kWarps][Sh::kRows], s_unit[Sh::kRows];
    __shared__ float2 s_ml[Sh::kRows];                  // this block's maximum and sum, for the cluster
    uint4* s_q = reinterpret_cast<uint4*>(dsm + kWarps * Sh::kPerWarp);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, tq = lane & 3;
    const int split = blockIdx.x, head = blockIdx.y / (uint32_t)a.tiles, r0 = (blockIdx.y - head * a.tiles) * Sh::kRows, m = blockIdx.z;
    pdl_trigger();
    pdl_wait();
    const int first = a.first[m], nodes = node_count(a, m);
    if (first < 0 || r0 >= nodes * a.group) return;     // (all blocks of the cluster)
    const int ctx = min(first, a.c.max_seq), end = (int)min((long)first + nodes, (long)a.c.max_seq);
    const int ntile = (end + kTile - 1) / kTile;
    const int each = ntile / (uint32_t)a.nsplit, over = ntile - each * a.nsplit;   // equal shares, the first ones a tile longer
    const int tile0 = split * each + min(split, over), tile1 = tile0 + each + (split < over ? 1 : 0);

    const size_t row0 = a.c.row(m, head, 0);
    constexpr int kRowBytes = kCoded ? kHd : 2 * kHd, kChunks = kRowBytes / 16, kStep = 32 / kChunks;
    const unsigned char *Kb = a.c.k + row0 * kRowBytes, *Vb = a.c.v + row0 * kRowBytes;
    const uint32_t stage0 = smem_u32(dsm + warp * Sh::kPerWarp);
    // masks of all nodes, for what nobody sees; only where this block comes to the nodes
    unsigned long long any = 0;
    const bool comes = tile1 * kTile > ctx;
    if (comes) {
        const unsigned long long mine = (lane < nodes ? mask_of(a, m, lane, nodes) : 0) | (lane + 32 < nodes ? mask_of(a, m, lane + 32, nodes) : 0);
        any = (unsigned long long)__reduce_or_sync(0xffffffffu, (uint32_t)(mine >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)mine);
        for (int r = t; r < Sh::kRows; r += kWarps * 32) s_mask[r] = r0 + r < nodes * a.group ? mask_of(a, m, (uint32_t)(r0 + r) / (uint32_t)a.group, nodes) : 0;
    }
    auto there = [&](int p) { return p < ctx || (p < end && (any >> (p - ctx) & 1)); };
    // 16 rows of K and V to a stage: piece c of rows rr, rr + kStep, ...; rows that nobody sees become zeros, whatever lies there
    const int c = lane % kChunks, rr = lane / kChunks;
    const uint32_t off = rr * kRowBytes + ((c ^ (rr & 7)) << 4);
    const float* scale = kCoded ? (lane < kTile ? a.c.ks : a.c.vs) + row0 + (lane & (kTile - 1)) : nullptr;
    auto issue = [&](int tile, int stage) {
        const int p0 = tile * kTile;
        const uint32_t to = stage0 + stage * Sh::kStage;
        const unsigned char *k = Kb + (size_t)(p0 + rr) * kRowBytes + c * 16, *v = Vb + (size_t)(p0 + rr) * kRowBytes + c * 16;
        if (p0 + kTile <= ctx) {
#pragma unroll
            for (int i = 0; i < kTile / kStep; ++i) {
                // the row's low bits: rr + kStep * i, of which kStep * i flips whole bits above rr's
                const uint32_t at = to + (off ^ (((kStep * i) & 7) << 4)) + kStep * i * kRowBytes;
                amma::cp_async16(at, k + i * kStep * kRowBytes);
                amma::cp_async16(at + Sh::kSide, v + i * kStep * kRowBytes);
            }
            if (kCoded) cp_async4z(to + 2 * Sh::kSide + lane * 4, scale + p0, true);
        } else {
#pragma unroll 1
            for (int i = 0; i < kTile / kStep; ++i) {
                const bool in = there(p0 + rr + kStep * i);
                const uint32_t at = to + (off ^ (((kStep * i) & 7) << 4)) + kStep * i * kRowBytes;
                lm::cp_async16z(at, in ? k + i * kStep * kRowBytes : Kb, in);
                lm::cp_async16z(at + Sh::kSide, in ? v + i * kStep * kRowBytes : Vb, in);
            }
            if (kCoded) {
                const bool in = there(p0 + (lane & (kTile - 1)));
                cp_async4z(to + 2 * Sh::kSide + lane * 4, scale + (in ? p0 : -(lane & (kTile - 1))), in);   // (the head's first row: in the cache, however short)
            }
        }
    };
    int next = tile0 + warp;
#pragma unroll
    for (int i = 0; i < Sh::kStages - 1; ++i) {
        if (next < tile1) issue(next, i);
        lm::cp_async_commit();
        next += kWarps;
    }

    // The query operand: column n of tile j is row r0 + 8 j + n.  Coded keys: a thread's four dimensions of k-step s are 32 tq + 4 s ...,
    // as it finds them in 16 bytes of a key row; otherwise 16 s + 2 tq, + 1, + 8, + 9.  Warp j brings tile j to its place, four lanes a row (each
    // warp fetching its operand by itself takes 256 lines of the cache a warp: 2,000 cycles with eight).
    constexpr float kScore = 0.08838834764831845f * 1.4426950408889634f;
    if (warp < NT) {
        const int r = 8 * warp + g, row = r0 + r, node = (uint32_t)row / (uint32_t)a.group;
        const bool in = node < nodes;
        const A* q = static_cast<const A*>(a.q) + (((size_t)m * a.T + (in ? node : 0)) * a.nq + head * a.group + (in ? row - node * a.group : 0)) * kHd + 4 * tq;
        float4 x[8];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = in ? lm::load4(q + 16 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float2 unit = binade(top);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint4 f;
            amma::split_hi_lo(x[i].x * unit.y, x[i].y * unit.y, f.x, f.z);
            amma::split_hi_lo(x[i].z * unit.y, x[i].w * unit.y, f.y, f.w);
            if (kCoded) {                               // lane l's operand of k-step s lies at l ^ s: banks
                const int st = 4 * (i & 1) + tq;
                s_q[(st * NT + warp) * 32 + ((4 * g + (i >> 1)) ^ st)] = f;
            } else {
                uint32_t *p0 = reinterpret_cast<uint32_t*>(s_q + (i * NT + warp) * 32 + ((4 * g + 2 * (tq & 1)) ^ i)) + (tq >> 1),
                         *p1 = reinterpret_cast<uint32_t*>(s_q + (i * NT + warp) * 32 + ((4 * g + 2 * (tq & 1) + 1) ^ i)) + (tq >> 1);
                p0[0] = f.x; p0[2] = f.z;
                p1[0] = f.y; p1[2] = f.w;
            }
        }
        if (tq == 0) s_unit[r] = unit.x * kScore;
    }
    __syncthreads();                                    // masks, queries
    constexpr int kRegs = NT > 2 ? 1 : NT;
    uint32_t qh[kRegs][8][2], ql[kSplit ? kRegs : 1][8][2];
    if (NT <= 2) {
#pragma unroll
        for (int j = 0; j < kRegs; ++j)
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const uint4 f = s_q[(st * NT + j) * 32 + ((kPair ? lane & 15 : lane) ^ st)];
                const bool low = kPair && lane > 15;
                qh[j][st][0] = low ? f.z : f.x; qh[j][st][1] = low ? f.w : f.y;
                if (kSplit) { ql[kSplit ? j : 0][st][0] = f.z; ql[kSplit ? j : 0][st][1] = f.w; }
            }
    }
    float qf[NT][2];                                    // factor of the scores of columns 2 tq, 2 tq + 1, base 2
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) qf[j][e] = s_unit[8 * j + ((2 * tq + e) & kRowOf)];

    float o[NT][8][4], mx[NT][2], l[NT][2], vunit = 1.f, vcap = -1.f, slack = kSlack;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        mx[j][0] = mx[j][1] = -FLT_MAX;
        l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[j][d][0] = o[j][d][1] = o[j][d][2] = o[j][d][3] = 0.f;
    }

    int stage = 0;
    for (int tile = tile0 + warp; tile < tile1; tile += kWarps) {
        if (next < tile1) issue(next, stage == 0 ? Sh::kStages - 1 : stage - 1);
        lm::cp_async_commit();
        next += kWarps;
        lm::cp_async_wait<Sh::kStages - 1>();
        __syncwarp();
        const uint32_t ks = stage0 + stage * Sh::kStage, vs = ks + Sh::kSide;
        float sc[4];                                    // scales of the keys g, g + 8 and of these values
        if (kCoded) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[e] = lds_f32(ks + 2 * Sh::kSide + ((e >> 1) * kTile + g + 8 * (e & 1)) * 4);
        }

        // ---- S^T: rows g, g + 8 of the tile's positions, columns 2 tq, 2 tq + 1 of each query tile
        float s[NT][4], s2[kSplit ? NT : 1][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
            if (kSplit) s2[j][0] = s2[j][1] = s2[j][2] = s2[j][3] = 0.f;
        }
        auto key_step = [&](int st, const uint32_t (&k)[4]) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (NT > 2) {
                    const uint4 b = s_q[(st * NT + j) * 32 + (lane ^ st)];
                    mma_f16(s[j], k, b.x, b.y);
                    if (kSplit) mma_f16(s2[kSplit ? j : 0], k, b.z, b.w);
                } else {
                    mma_f16(s[j], k, qh[NT > 2 ? 0 : j][st][0], qh[NT > 2 ? 0 : j][st][1]);
                    if (kSplit) mma_f16(s2[kSplit ? j : 0], k, ql[NT > 2 || !kSplit ? 0 : j][st][0], ql[NT > 2 || !kSplit ? 0 : j][st][1]);
                }
            }
        };
        if (kCoded) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {            // 16 bytes: four k-steps
                uint4 lo, hi;
                const uint32_t at = ks + g * kHd + (((2 * tq + hf) ^ g) << 4);
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w) : "r"(at));
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w) : "r"(at + 8 * kHd));
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t k[4];
                    codes_f16(wl[e], k[0], k[2]);
                    codes_f16(wh[e], k[1], k[3]);
                    key_step(4 * hf + e, k);
                }
            }
        } else {
            const int mi = lane >> 3, r8 = lane & 7;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                uint32_t k[4];
                amma::ldmatrix_x4(ks + ((mi & 1) * 8 + r8) * 2 * kHd + (((2 * st + (mi >> 1)) ^ r8) << 4), k[0], k[1], k[2], k[3]);
                key_step(st, k);
            }
        }
        // ---- scores in base 2; masks where the tile reaches the nodes
        const int p0 = tile * kTile;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = s[j][e];
                if (kSplit) x += s2[kSplit ? j : 0][e];
                if (kPair) x += __shfl_xor_sync(0xffffffffu, x, 2);
                x *= qf[j][e & 1];
                if (kCoded) x *= sc[e >> 1];
                s[j][e] = x;
            }
        if (p0 + kTile > ctx) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int p = p0 + g + 8 * (e >> 1);
                    const bool yes = p < ctx || (p < end && (s_mask[8 * j + ((2 * tq + (e & 1)) & kRowOf)] >> (p - ctx) & 1));
                    s[j][e] = yes ? s[j][e] : -INFINITY;
                }
        }
        // Codes: a score is compared beside a cap of the value scales that the lane multiplies with, set anew when one exceeds it or the reference
        // moves: to four times the present one or more, at most 2^8 times (2^(kSlack - kHead): a cap up to there hardly moves a reference in vain;
        // scales up to 2^8 apart cost 1 to 2 %, where a cap of four times the last one cost 8 to 16).
        bool move = kCoded && fmaxf(fabsf(sc[2]), fabsf(sc[3])) > vcap;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) move |= fmaxf(s[j][e], s[j][e + 2]) > mx[j][e] + slack;
        if (__any_sync(0xffffffffu, move)) {
            float lg[2] = {0.f, 0.f};
            if (kCoded) {
                const float top = fmaxf(fabsf(sc[2]), fabsf(sc[3])), unit = scale_unit(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                vunit = tile == tile0 + warp ? unit : vunit;     // (the first tile comes here)
                const float vdiv = __uint_as_float((254u << 23) - __float_as_uint(vunit));
                lg[0] = scale_log2(sc[2] * vdiv);
                lg[1] = scale_log2(sc[3] * vdiv);
                vcap = fmaxf(4.f * top, fminf(vcap, 256.f * top));
                slack = kSlack - scale_log2(vcap * vdiv);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[j][e] + lg[0], s[j][e + 2] + lg[1]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float to = fmaxf(mx[j][e], top - kHead);
                    const float2 h = step<kCoded>(mx[j][e], to);
                    mx[j][e] = to;
                    l[j][e] = l[j][e] * h.x * h.y;
                    f[e] = h.x * h.y;
                }
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    o[j][d][0] *= f[0]; o[j][d][1] *= f[1];
                    o[j][d][2] *= f[0]; o[j][d][3] *= f[1];
                }
            }
        }
        // ---- P^T, and to the operand layout
        if (kCoded) {
            const float vdiv = __uint_as_float((254u << 23) - __float_as_uint(vunit));
            sc[2] *= vdiv;
            sc[3] *= vdiv;
        }
        uint32_t ph[NT][2], pl[kSplit ? NT : 1][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = lm::exp2_fast(s[j][e] - mx[j][e & 1]);
                l[j][e & 1] += p[e];
                if (kCoded) p[e] *= sc[2 + (e >> 1)];
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (kSplit) {
                    uint32_t h, lo;
                    amma::split_hi_lo(p[2 * e], p[2 * e + 1], h, lo);
                    ph[j][e] = transpose8x8(h);
                    pl[kSplit ? j : 0][e] = transpose8x8(lo);
                } else if (kPair) {
                    uint32_t h, lo;
                    amma::split_hi_lo(p[2 * e], p[2 * e + 1], h, lo);
                    ph[j][e] = transpose8x8(tq < 2 ? h : lo);
                } else {
                    const __half2 h = __floats2half2_rn(p[2 * e], p[2 * e + 1]);
                    ph[j][e] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
                }
            }
        }
        // ---- O^T += V^T P^T.  Coded values: rows g / g + 8 of dimension tile d are dimensions 16 g + 2 d / + 1, 16 bytes of a value row.
        auto value_step = [&](int d, const uint32_t (&v)[4]) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (kSplit) {
                    float c[4];
                    mma_f16_new(c, v, pl[kSplit ? j : 0][0], pl[kSplit ? j : 0][1]);
                    mma_f16(c, v, ph[j][0], ph[j][1]);
                    add2(o[j][d][0], o[j][d][1], c[0], c[1]);
                    add2(o[j][d][2], o[j][d][3], c[2], c[3]);
                } else if (kPair) {
                    float c[4];
                    mma_f16_new(c, v, ph[j][0], ph[j][1]);
                    add2(o[j][d][0], o[j][d][1], c[0], c[1]);
                    add2(o[j][d][2], o[j][d][3], c[2], c[3]);
                } else {
                    mma_f16(o[j][d], v, ph[j][0], ph[j][1]);
                }
            }
        };
        if (kCoded) {
            uint4 w[4];                                 // positions 2 tq, + 1, + 8, + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * tq + (i & 1) + 8 * (i >> 1);
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                             : "r"(vs + r * kHd + ((g ^ (r & 7)) << 4)));
            }
#pragma unroll
            for (int d = 0; d < 8; d += 2) {
                const uint32_t x[4] = {d < 2 ? w[0].x : d < 4 ? w[0].y : d < 6 ? w[0].z : w[0].w, d < 2 ? w[1].x : d < 4 ? w[1].y : d < 6 ? w[1].z : w[1].w,
                                       d < 2 ? w[2].x : d < 4 ? w[2].y : d < 6 ? w[2].z : w[2].w, d < 2 ? w[3].x : d < 4 ? w[3].y : d < 6 ? w[3].z : w[3].w};
#pragma unroll
                for (int e = 0; e < 2; ++e) {           // bytes 2 e, 2 e + 1 of two positions: b0 b0' b1 b1'
                    uint32_t v[4];
                    codes_f16(prmt(x[0], x[1], e ? 0x7362 : 0x5140), v[0], v[1]);
                    codes_f16(prmt(x[2], x[3], e ? 0x7362 : 0x5140), v[2], v[3]);
                    value_step(d + e, v);
                }
            }
        } else {
            const int mi = lane >> 3, r8 = lane & 7;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                uint32_t v[4];
                amma::ldmatrix_x4_trans(vs + ((mi >> 1) * 8 + r8) * 2 * kHd + (((2 * d + (mi & 1)) ^ r8) << 4), v[0], v[1], v[2], v[3]);
                value_step(d, v);
            }
        }
        __syncwarp();                                   // the stage is filled again in the next turn
        stage = stage == Sh::kStages - 1 ? 0 : stage + 1;
    }
    lm::cp_async_wait<0>();
    __syncwarp();

    // ---- the warps' results to shared memory: [row][128]
    float* so = reinterpret_cast<float*>(dsm + warp * Sh::kPerWarp);
    if (kPair) {                                        // high parts and remainders: lanes of columns 0-3 get dimension tiles 0-3, the others 4-7
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float mine = tq < 2 ? o[0][d][e] : o[0][d + 4][e], other = tq < 2 ? o[0][d + 4][e] : o[0][d][e];
                o[0][d][e] = mine + __shfl_xor_sync(0xffffffffu, other, 2);
            }
    }
    constexpr int kTiles = kPair ? 4 : 8;
    const int d0 = kPair && tq > 1 ? 4 : 0;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[j][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int r = 8 * j + ((2 * tq + e) & kRowOf);
            if (g == 0) { s_m[warp][r] = mx[j][e]; s_l[warp][r] = sum; }
#pragma unroll
            for (int d = 0; d < kTiles; ++d) {
                if (kCoded) {
                    *reinterpret_cast<float2*>(so + r * kHd + 16 * g + 2 * (d0 + d)) = make_float2(o[j][d][e] * vunit, o[j][d][e + 2] * vunit);
                } else {
                    so[r * kHd + 16 * (d0 + d) + g] = o[j][d][e];
                    so[r * kHd + 16 * (d0 + d) + g + 8] = o[j][d][e + 2];
                }
            }
        }
    __syncthreads();
    // ---- and together: a warp per row, four dimensions a lane; over the first warp's where a cluster goes on with them
    const int groups = a.nsplit / a.cluster, grp = split / a.cluster;
    auto emit = [&](int r, const float4& acc, float top, float sum) {
        const int row = r0 + r, node = (uint32_t)row / (uint32_t)a.group;
        if (groups == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // a row that sees nothing: 0
            A* out = static_cast<A*>(a.out) + (((size_t)m * a.T + node) * a.nq + head * a.group + row - node * a.group) * kHd + 4 * lane;
            lm::store4(out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        } else {
            float* rec = a.part + ((((size_t)m * a.c.heads + head) * a.rows + row) * groups + grp) * kPart;
            *reinterpret_cast<float4*>(rec + 4 * lane) = acc;
            if (lane == 0) *reinterpret_cast<float2*>(rec + kHd) = make_float2(top, sum);
        }
    };
    const int rows = min(Sh::kRows, nodes * a.group - r0);
    for (int r = warp; r < rows; r += kWarps) {
        float top = -FLT_MAX, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 h = step<kCoded>(s_m[w][r], top);
            const float cc = h.x * h.y;
            const float4 v = *reinterpret_cast<const float4*>(dsm + w * Sh::kPerWarp + (r * kHd + 4 * lane) * 4);
            sum = fmaf(s_l[w][r] * h.y, h.x, sum);
            acc.x = fmaf(v.x, cc, acc.x); acc.y = fmaf(v.y, cc, acc.y); acc.z = fmaf(v.z, cc, acc.z); acc.w = fmaf(v.w, cc, acc.w);
        }
        if (a.cluster == 1) {
            emit(r, acc, top, sum);
        } else {
            *reinterpret_cast<float4*>(dsm + (r * kHd + 4 * lane) * 4) = acc;   // (this lane alone reads and writes there)
            if (lane == 0) s_ml[r] = make_float2(top, sum);
        }
    }
    if (a.cluster == 1) return;
    cluster_sync_all();                                 // every block's record is in its shared memory
    const int rank = split - grp * a.cluster;
    for (int r = rank + warp * a.cluster; r < rows; r += kWarps * a.cluster) {
        const uint32_t ml = smem_u32(&s_ml[r]), ov = smem_u32(dsm) + (r * kHd + 4 * lane) * 4;
        const bool has = lane < a.cluster;
        const float tb = has ? ld_dsmem(ml, lane) : -FLT_MAX, lb = has ? ld_dsmem(ml + 4, lane) : 0.f;
        const float top = warp_max(tb);
        const float2 h = step<kCoded>(tb, top);
        const float wgt = h.x * h.y, sum = warp_sum(lb * h.x * h.y);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int b = 0; b < a.cluster; ++b) {
            const float cc = __shfl_sync(0xffffffffu, wgt, b);
            const float4 v = ld_dsmem4(ov, b);
            acc.x = fmaf(v.x, cc, acc.x); acc.y = fmaf(v.y, cc, acc.y); acc.z = fmaf(v.z, cc, acc.z); acc.w = fmaf(v.w, cc, acc.w);
        }
        emit(r, acc, top, sum);
    }
    cluster_sync_all();                                 // nobody leaves while its record may still be read
}

// The clusters' records of a row, a warp each.
template <typename A>
__global__ void __launch_bounds__(128) attend_merge_kernel(const Args a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 5);     // (m, head, row)
    if (at >= (long)a.M * a.c.heads * a.rows) return;
    const int row = (int)(at % a.rows), mh = (int)(at / a.rows), m = mh / a.c.heads, head = mh - m * a.c.heads, node = row / a.group;
    if (a.first[m] < 0 || node >= node_count(a, m)) return;
    const int parts = a.nsplit / a.cluster;
    const float* rec = a.part + (size_t)at * parts * kPart;
    float top = -FLT_MAX, sum = 0.f;
    for (int s = lane; s < parts; s += 32) top = fmaxf(top, rec[(size_t)s * kPart + kHd]);
    top = warp_max(top);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(rec + (size_t)s * kPart + kHd);
        const float4 v = *reinterpret_cast<const float4*>(rec + (size_t)s * kPart + 4 * lane);
        const float2 h = step<true>(ml.x, top);
        const float c = h.x * h.y;
        sum = fmaf(ml.y * h.y, h.x, sum);
        acc.x = fmaf(v.x, c, acc.x); acc.y = fmaf(v.y, c, acc.y); acc.z = fmaf(v.z, c, acc.z); acc.w = fmaf(v.w, c, acc.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    A* out = static_cast<A*>(a.out) + (((size_t)m * a.T + node) * a.nq + head * a.group + row - node * a.group) * kHd + 4 * lane;
    lm::store4(out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

}  // namespace tree
}  // namespace bw
