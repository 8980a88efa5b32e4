// The same attention on the 5th-generation tensor cores.
//
// One block of 512 threads per SM.  Query rows (node, query head of the group) are the 128 lanes of an accumulator; two accumulator sets
// ("streams") keep the tensor cores busy while the softmax of one runs:
//   kTall   more than 128 rows: each stream has 128 rows, both take every 64 positions of the context
//   else    each stream has all rows and takes every other 64 positions; at the end they join what they have, half of the columns each
// Warps 0-3 and 4-7: softmax of a stream, a thread per row.  Warps 8-11: the cache; binary16 rows go to their swizzled place by cp.async, codes
// come raw, become f16 (exact) and are stored there.  Warps 12 and 13 issue a stream's products each:
//   S = Q K^T    two S buffers of 64 columns per stream, the next scores are on their way while the softmax has these
//   O += P V     P over the scores' columns as the f16 A operand, V from shared memory as it lies there ([position][column])
// fp32 activations: Q and P as f16 high parts and remainders, multiplied one after the other.  The accumulator's sums are cut, not rounded, at
// 24 bits, which adds up: so the remainders of a score come first, and O is added to a sum in the scratch memory (L2) every four tiles and
// starts afresh (57 nodes over 5,279 positions: error 1.1e-6 of the result, as that of 32-bit sums; every eight tiles 2.3e-6 and a tenth faster).
// Scales and the moving reference as in attention_tree.cuh (scales relative to the size of a part's first); a warp brings its rows of O to a new one by itself.
// Work is shared out in tiles of 64 positions: all sequences' tiles, heads and row groups in one line, an equal stretch of it per block; what
// a block has of a head's context that it does not have whole goes to a record that the merge kernel joins.
// All waits are bounded; a wait that gives up raises an abort flag.
// Measured (8 trees of 64 nodes over 2,000 to 4,096 positions, 32 / 8 heads, 8 bits): bf16 57 us, 0.43 PFLOP/s, fp32 92.5.  Of a block's 85,000 cycles a
// tile takes 2,600, the softmax of a stream that long from one tile to the next (scores out of tensor memory 250, scales and maximum 600, exponentials 1,200;
// the units' own rates would allow 1,100, the rest is latency of one warp per scheduler and stream); the start 4,000, and each of two parts 10,000 to
// 12,000 for the queries' place, the first scores and the record of 128 KB (stored a column at a time it took 5,000).  The merge takes 5 us.  Tried and not kept: maximum and exponentials in
// one pass over the scores (slower), streams held half a tile apart (1 to 3 %).
#pragma once
#include "attention_tree.cuh"
#include "gemm_w4a8_tc.cuh"

namespace bw {
namespace tree {

constexpr int kTcKeys = 64, kTcPanel = kTcKeys * 128, kTcThreads = 512;   // positions of a tile, bytes of 64 x 64 f16
constexpr int kTcStage = 4 * kTcPanel;                                    // K and V of a tile
constexpr int kTcRaw = 2 * kTcKeys * kHd + 2 * kTcKeys * 4;               // codes and scales of a tile
constexpr int kFlush = 4;
constexpr float kNear = 4.f;                                               // value scales of a tile up to 2^4 apart are of one size
constexpr int kPlanned = 448;                                              // sequences whose work is laid out in a line

template <bool kTall, bool kCoded, bool kSplit>
struct TcShape {
    static constexpr int kQTile = 4 * kTcPanel;                                      // 128 rows x 128
    static constexpr int kQ = (kTall ? 2 : 1) * (kSplit ? 2 : 1) * kQTile;
    static constexpr int kStages = kTall && kSplit ? 2 : kCoded ? 3 : 4;
    static constexpr int kRaws = !kCoded ? 0 : kTall && kSplit ? 1 : kTall || kSplit ? 3 : 4;
    static constexpr int kHead = 14848;                                              // barriers, the line of work, what stream 1 hands over
    static constexpr int kScales = (kHead + kStages * 2 * kTcKeys * 4 + 1023) / 1024 * 1024 - kHead;
    static constexpr int kSmem = 1024 + kHead + kScales + kQ + kStages * kTcStage + kRaws * kTcRaw;
    static_assert(kSmem <= 232448, "shared memory of a block");
    // registers per thread: 256 softmax threads, 256 others; 65,536 together, what 512 threads of 128 start with
    static constexpr int kRegsSoftmax = 168, kRegsOther = 256 - kRegsSoftmax;
    // barriers
    static constexpr int kFullQ = 0, kFullS = 1, kFullP = 5, kDoneO = 9, kDrain = 13, kGive = 14, kTaken = 15, kFullKV = 16,
                         kEmptyKV = kFullKV + kStages, kBars = kEmptyKV + kStages;
};

// ------------------------------------------------------------------------------------------------------------------ work in a line
struct Seq {
    int first, nodes, tiles, groups;    // tiles of 64 positions, row groups; none: 0
};
__device__ __forceinline__ Seq seq_of(const Args& a, int m) {
    Seq s{a.first[m], node_count(a, m), 0, 0};
    if (s.first >= 0 && s.nodes > 0) {
        s.tiles = ((int)min((long)s.first + s.nodes, (long)a.c.max_seq) + kTcKeys - 1) / kTcKeys;
        s.groups = (s.nodes * a.group + a.group_rows - 1) / a.group_rows;
    }
    return s;
}
struct Part {
    int m, head, group, t0, t1, slot;   // slot < 0: the head's whole context
    int first, nodes;
};

// (x, y) *= (fx, fy), as one instruction.
__device__ __forceinline__ void mul2(float& x, float& y, float fx, float fy) {
    asm("{\n\t.reg .b64 v, f;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 f, {%2, %3};\n\tmul.rn.f32x2 v, v, f;\n\tmov.b64 {%0, %1}, v;\n\t}" : "+f"(x), "+f"(y) : "f"(fx), "f"(fy));
}
// (x, y) = (x, y) * f + c, as one instruction.
__device__ __forceinline__ void fma2(float& x, float& y, float f, float c) {
    asm("{\n\t.reg .b64 v, f, c;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 f, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\tfma.rn.f32x2 v, v, f, c;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y) : "f"(f), "f"(c));
}
// f16 high parts and remainders of a pair.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    add2(x, y, -f.x, -f.y);
    const __half2 l = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void mul2(uint32_t& x, uint32_t& y, float fx, float fy) {
    float a = __uint_as_float(x), b = __uint_as_float(y);
    mul2(a, b, fx, fy);
    x = __float_as_uint(a);
    y = __float_as_uint(b);
}

__device__ __forceinline__ void store_o16(float* p, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
__device__ __forceinline__ void store_o16(__nv_bfloat16* p, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(lm::pack_bf16(v[8 * i], v[8 * i + 1]), lm::pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                                                    lm::pack_bf16(v[8 * i + 4], v[8 * i + 5]), lm::pack_bf16(v[8 * i + 6], v[8 * i + 7]));
}

template <bool kTall, bool kCoded, typename A>
__global__ void __launch_bounds__(kTcThreads, 1) attend_tc_kernel(const Args a) {
    constexpr bool kSplit = sizeof(A) == 4;
    using Sh = TcShape<kTall, kCoded, kSplit>;
    constexpr int NS = Sh::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023);   // (not rounded as an address: loads stay loads of shared memory)
    unsigned char* q_area = smem + Sh::kHead + Sh::kScales;       // (a multiple of 1,024 from the base)
    static_assert((Sh::kHead + Sh::kScales) % 1024 == 0, "swizzled tiles start at 1,024 bytes");
    const uint32_t sq = smem_u32(q_area), skv = sq + Sh::kQ, sraw = skv + NS * kTcStage, bar0 = smem_u32(smem), flag = bar0 + 516;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 516);
    int* s_cum = reinterpret_cast<int*>(smem + 768);               // [kPlanned]: tiles of all sequences before
    Seq* s_seq = reinterpret_cast<Seq*>(smem + 2560);              // [kPlanned]
    float4* s_ml = reinterpret_cast<float4*>(smem + 9728);         // [2][128] maximum, sum, scales that a stream shows the other
    float* s_qf = reinterpret_cast<float*>(smem + 13824);          // [128] factors of the rows that both streams have
    static_assert(768 + kPlanned * 4 <= 2560 && 2560 + kPlanned * sizeof(Seq) <= 9728 && 9728 + 4096 <= 13824 && 13824 + 512 <= Sh::kHead, "layout");
    float* s_scale = reinterpret_cast<float*>(smem + Sh::kHead);   // [stage][K 64, V 64]
    // [stage]: what the part's value scales are relative to; log2 of the tile's largest, and of its smallest
    float *s_unit = reinterpret_cast<float*>(smem + 520), *s_top = reinterpret_cast<float*>(smem + 536), *s_low = reinterpret_cast<float*>(smem + 552);
    const int t = threadIdx.x, warp = __shfl_sync(0xffffffffu, t >> 5, 0), lane = t & 31;
    auto bar = [&](int i) { return bar0 + 8 * i; };
    auto wait = [&](int i, uint32_t parity) { mbar_wait_or_abort(bar(i), parity, flag); };
    if (t == 0) {
        mbar_init(bar(Sh::kFullQ), 256);
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(Sh::kFullS + i), 1);
            mbar_init(bar(Sh::kFullP + i), 4);
            mbar_init(bar(Sh::kDoneO + i), 1);
        }
        mbar_init(bar(Sh::kDrain), 2);
        mbar_init(bar(Sh::kGive), 256);
        mbar_init(bar(Sh::kTaken), 256);
        for (int i = 0; i < NS; ++i) {
            mbar_init(bar(Sh::kFullKV + i), 128);
            mbar_init(bar(Sh::kEmptyKV + i), kTall ? 2 : 1);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 12) {
        tc::tmem_alloc(bar0 + 512, 512);
        tc::tmem_relinquish();
    }
    pdl_trigger();
    pdl_wait();
    // ---- the line of work: tiles of the sequences before each
    int line = 0;
    if (a.flat) {
        int* s_warp = reinterpret_cast<int*>(smem + 640);          // [16]
        int v = 0;
        if (t < a.M) {
            const Seq q = seq_of(a, t);
            s_seq[t] = q;
            v = q.tiles * q.groups * a.c.heads;
        }
        int sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        if (lane == 31) s_warp[warp] = sum;
        __syncthreads();
        int before = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int u = s_warp[w];
            before += w < warp ? u : 0;
            line += u;
        }
        if (t < a.M) s_cum[t] = before + sum - v;
        if (blockIdx.x == 0) {                                     // for the merge
            if (t < a.M) a.cum[t] = before + sum - v;
            if (t <= a.blocks) a.cum[kPlanned + t] = (int)((long)line * t / a.blocks);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(smem + 512), 0);
    const int c = blockIdx.x, x_first = a.flat ? (int)((long)line * c / a.blocks) : c, x_end = a.flat ? (int)((long)line * (c + 1) / a.blocks) : a.pairs;
    // Part number 0, 1, ... of this block: false after the last.  x: where it starts in the line, moved on; without a line, the number of a
    // sequence's head and row group, every blocks-th of which is this block's, whole.
    auto next_part = [&](int& x, Part& p) {
        if (x >= x_end) return false;
        if (a.flat) {
            int lo = 0, hi = a.M - 1;                              // the last sequence that starts at or before x
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_cum[mid] <= x) lo = mid; else hi = mid - 1;
            }
            const Seq q = s_seq[lo];
            const uint32_t rel = x - s_cum[lo], pair = rel / (uint32_t)q.tiles;
            p.m = lo;
            p.first = q.first;
            p.nodes = q.nodes;
            p.head = q.groups == 1 ? pair : pair / (uint32_t)q.groups;
            p.group = pair - p.head * q.groups;
            p.t0 = rel - pair * q.tiles;
            p.t1 = min(q.tiles, p.t0 + x_end - x);
            p.slot = p.t0 == 0 && p.t1 == q.tiles ? -1 : 2 * c + (x == x_first ? 0 : 1);
            x += p.t1 - p.t0;
            return true;
        }
        for (; x < x_end; x += a.blocks) {
            const uint32_t mh = x / (uint32_t)a.groups;
            p.group = x - mh * a.groups;
            p.m = mh / (uint32_t)a.c.heads;
            p.head = mh - p.m * a.c.heads;
            const Seq q = seq_of(a, p.m);
            if (p.group >= q.groups) continue;
            p.first = q.first;
            p.nodes = q.nodes;
            p.t0 = 0;
            p.t1 = q.tiles;
            p.slot = -1;
            x += a.blocks;
            return true;
        }
        return false;
    };
    // Jobs of a part for stream w: all its tiles (kTall), else tiles w, w + 2, ...

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::kRegsOther));
        if (warp < 14) {
            // A warp per stream; the whole warp walks the loop, one elected lane issues.  The scores of the next tile go out before this
            // tile's second product.
            constexpr uint32_t id_s = tc::idesc_f16(kTcKeys), id_o = tc::idesc_f16(kHd, true);
            const bool elected = tc::elect_one();
            const int w = warp - 12;
            const uint32_t acc = tmem + w * 256, q = sq + (kTall ? w : 0) * (kSplit ? 2 : 1) * Sh::kQTile;
            int x = x_first, kb = 0, nth = 0, st_s = 0, st_o = 0;  // stages of the next scores, of the next second product
            uint32_t lap = 0;                                      // parity of the next scores' stage
            Part p;
            auto walk = [&](int by) {
                st_s += by;
                if (st_s >= NS) {
                    st_s -= NS;
                    lap ^= 1;
                }
            };
            for (; next_part(x, p) && !*abort_flag; ++nth) {
                const int tiles = p.t1 - p.t0, jobs = kTall ? tiles : (tiles + 1 - w) >> 1;
                auto scores = [&](int k) {
                    const int kk = kb + k, b = kk & 1;
                    if (kk > 1) wait(Sh::kDoneO + 2 * w + b, ((kk - 2) >> 1) & 1);   // the P that lay there has been multiplied
                    wait(Sh::kFullKV + st_s, lap);
                    tc::tc_fence_after();
                    if (elected) {
                        const uint32_t d = acc + b * 64, kt = skv + st_s * kTcStage;
#pragma unroll
                        for (int part = kSplit ? 1 : 0; part >= 0; --part)   // remainders first, while the sum is small
#pragma unroll
                            for (int pan = 0; pan < 2; ++pan)
#pragma unroll
                                for (int e = 0; e < 4; ++e)   // 16 dimensions = 32 bytes further inside the swizzle atom
                                    tc::tc_mma_bf16(d, tc::flash_desc(q + part * Sh::kQTile + pan * 2 * kTcPanel, 16, 1024) + 2 * e,
                                                    tc::flash_desc(kt + pan * kTcPanel, 16, 1024) + 2 * e, id_s, part < (kSplit ? 1 : 0) || pan + e > 0 ? 1u : 0u);
                        tc::tc_commit(bar(Sh::kFullS + 2 * w + b));
                    }
                    __syncwarp();
                    walk(kTall ? 1 : 2);
                };
                if (!kTall && w == 1) walk(1);
                st_o = st_s;
                wait(Sh::kFullQ, nth & 1);
                tc::tc_fence_after();
                if (jobs > 0) scores(0);
                for (int k = 0; k < jobs && !*abort_flag; ++k) {
                    if (k + 1 < jobs) scores(k + 1);
                    const int kk = kb + k, b = kk & 1;
                    wait(Sh::kFullP + 2 * w + b, (kk >> 1) & 1);
                    tc::tc_fence_after();
                    if (elected) {
                        const uint32_t pa = acc + b * 64, o = acc + 128, v = skv + st_o * kTcStage + 2 * kTcPanel;
                        const bool fresh = kSplit ? k % kFlush == 0 : k == 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {   // 16 positions: two 8-row groups
                            const uint64_t vd = tc::flash_desc(v, kTcPanel, 1024) + e * (2048 >> 4);
                            const uint32_t at = pa + (kSplit ? 16 * e : (e >> 1) * 32 + (e & 1) * 8);
                            tc::tc_mma_bf16_ta(o, at, vd, id_o, fresh && e == 0 ? 0u : 1u);
                            if (kSplit) tc::tc_mma_bf16_ta(o, at + 8, vd, id_o, 1u);
                        }
                        tc::tc_commit(bar(Sh::kDoneO + 2 * w + b));
                        tc::tc_commit(bar(Sh::kEmptyKV + st_o));
                    }
                    __syncwarp();
                    st_o += kTall ? 1 : 2;
                    if (st_o >= NS) st_o -= NS;
                }
                // to the first stage after the part: a stream's scores stand behind its last tile and the next but one
                if (!kTall && jobs > 0 && ((tiles ^ w) & 1) == 1) {   // one too far
                    if (st_s == 0) lap ^= 1;
                    st_s = st_s == 0 ? NS - 1 : st_s - 1;
                }
                kb += jobs;
            }
            if (elected) tc::tc_commit(bar(Sh::kDrain));   // whatever became of the others: no MMA in flight when the tensor memory is freed
            __syncwarp();
            mbar_wait(bar(Sh::kDrain), 0);
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::kRegsOther));
        // ---- the cache, 128 threads: piece `pc` (16 bytes) of rows r0, r0 + 16 (codes) / r0 + 8 (binary16), ...
        const int u = t - 256, pc = kCoded ? u & 7 : u & 15, r0 = kCoded ? u >> 3 : u >> 4;
        constexpr int kStep = kCoded ? 16 : 8, kRows = kTcKeys / kStep, kRowBytes = kCoded ? kHd : 2 * kHd;
        // Tiles in flight.  The products free a tile's stage once the next tile (kTall) or the next but one is there: no more stages than
        // that leaves may be asked for ahead of it.
        constexpr int kAhead = kCoded ? Sh::kRaws : kTall ? NS - 1 : NS - 2;
        static_assert(NS >= (kTall ? 2 : 3) && kAhead >= 1, "stages");
        int x = x_first, it_in = 0, it_out = 0, st_in = 0, st_out = 0, raw_in = 0, raw_out = 0;
        uint32_t lap_in = 1, lap_out = 1;                          // parity of the stages' next release
        uint32_t opens = 0;                                        // of the tiles in flight, by number modulo 32: first of a part
        bool more, opening = false;
        int tile = 0, tile_end = 0, ctx = 0, end = 0;
        unsigned long long any = 0;
        size_t row0 = 0;
        auto open_part = [&]() {                                   // the next part and what its sequence's rows see
            Part p{};
            more = next_part(x, p);
            if (!more) return;
            opening = true;
            tile = p.t0;
            tile_end = p.t1;
            ctx = min(p.first, a.c.max_seq);
            end = (int)min((long)p.first + p.nodes, (long)a.c.max_seq);
            any = 0;
            if (tile_end * kTcKeys > ctx) {
                const unsigned long long mine = (lane < p.nodes ? mask_of(a, p.m, lane, p.nodes) : 0) | (lane + 32 < p.nodes ? mask_of(a, p.m, lane + 32, p.nodes) : 0);
                any = (unsigned long long)__reduce_or_sync(0xffffffffu, (uint32_t)(mine >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)mine);
            }
            row0 = a.c.row(p.m, p.head, 0);
        };
        open_part();
        // where this thread's piece of row r0 goes; the others are kStep rows on (binary16: swizzled, kStep = 8 keeps a row's low bits)
        const uint32_t place = kCoded ? r0 * kHd + pc * 16 : (pc >> 3) * kTcPanel + r0 * 128 + (((pc & 7) ^ (r0 & 7)) << 4);
        constexpr uint32_t kSideOff = kCoded ? kTcKeys * kHd : 2 * kTcPanel, kRowOff = kStep * 128;
        auto issue = [&]() {                                       // the next tile on its way
            if (more) {
                const int p0 = tile * kTcKeys;
                if (!kCoded) wait(Sh::kEmptyKV + st_in, lap_in);
                const uint32_t to = kCoded ? sraw + raw_in * kTcRaw : skv + st_in * kTcStage;
                const size_t first_row = (row0 + p0 + r0) * kRowBytes + pc * 16;
                const unsigned char *k = a.c.k + first_row, *v = a.c.v + first_row;
                if (p0 + kTcKeys <= ctx) {
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        amma::cp_async16(to + place + i * kRowOff, k + i * kStep * kRowBytes);
                        amma::cp_async16(to + place + kSideOff + i * kRowOff, v + i * kStep * kRowBytes);
                    }
                    if (kCoded && (warp & 1) == 0) {               // warp 8 the keys' scales, warp 10 the values'
                        const float* f = (warp == 8 ? a.c.ks : a.c.vs) + row0 + p0 + lane;
                        tc::cp_async4(to + 2 * kTcKeys * kHd + (warp - 8) * 128 + lane * 4, f, 4);
                        tc::cp_async4(to + 2 * kTcKeys * kHd + (warp - 8) * 128 + 128 + lane * 4, f + 32, 4);
                    }
                } else {
                    auto there = [&](int p) { return p < ctx || (p < end && (any >> (p - ctx) & 1)); };
#pragma unroll 1
                    for (int i = 0; i < kRows; ++i) {
                        const bool in_seq = there(p0 + r0 + kStep * i);
                        lm::cp_async16z(to + place + i * kRowOff, in_seq ? k + i * kStep * kRowBytes : a.c.k, in_seq);
                        lm::cp_async16z(to + place + kSideOff + i * kRowOff, in_seq ? v + i * kStep * kRowBytes : a.c.v, in_seq);
                    }
                    if (kCoded && (warp & 1) == 0) {
#pragma unroll 1
                        for (int i = 0; i < 2; ++i) {
                            const int p = p0 + lane + 32 * i;
                            const bool in_seq = there(p);
                            tc::cp_async4(to + 2 * kTcKeys * kHd + (warp - 8) * 128 + 128 * i + lane * 4,
                                          (warp == 8 ? a.c.ks : a.c.vs) + row0 + (in_seq ? p : 0), in_seq ? 4 : 0);
                        }
                    }
                }
                opens = (opens & ~(1u << (it_in & 31))) | (opening ? 1u : 0u) << (it_in & 31);
                opening = false;
                ++it_in;
                if (kCoded) {
                    raw_in = raw_in == Sh::kRaws - 1 ? 0 : raw_in + 1;
                } else if (++st_in == NS) {
                    st_in = 0;
                    lap_in ^= 1;
                }
                if (++tile == tile_end) open_part();
            }
            lm::cp_async_commit();
        };
        float vunit = 1.f;                                         // warp 10: what the part's value scales are relative to
#pragma unroll
        for (int i = 0; i < kAhead; ++i) issue();
        while ((more || it_out < it_in) && !*abort_flag) {
            const int st = st_out;
            lm::cp_async_wait<kAhead - 1>();
            if (kCoded) {
                wait(Sh::kEmptyKV + st, lap_out);
                const uint32_t from = sraw + raw_out * kTcRaw, to = skv + st * kTcStage;
                if ((warp & 1) == 0) {
                    // The scales, by whom copied them.  A value's is given relative to the size of the part's first.
                    const float* fs = reinterpret_cast<const float*>(smem + (from - bar0) + 2 * kTcKeys * kHd) + (warp - 8) * 32 + lane;
                    float s0 = fs[0], s1 = fs[32];
                    if (warp == 10) {
                        const uint32_t b0 = __float_as_uint(fabsf(s0)), b1 = __float_as_uint(fabsf(s1)), top = __reduce_max_sync(0xffffffffu, max(b0, b1));
                        const uint32_t low = __reduce_min_sync(0xffffffffu, min(b0, b1));   // (0 in a tile with rows that nobody sees, too)
                        if (opens >> (it_out & 31) & 1) vunit = scale_unit(top);
                        const float inv = __uint_as_float((254u << 23) - __float_as_uint(vunit));
                        s0 *= inv;
                        s1 *= inv;
                        if (lane == 0) {
                            s_unit[st] = vunit;
                            s_top[st] = scale_log2(__uint_as_float(top) * inv);
                            s_low[st] = scale_log2(__uint_as_float(low) * inv);
                        }
                    }
                    s_scale[st * 2 * kTcKeys + (warp - 8) * 32 + lane] = s0;
                    s_scale[st * 2 * kTcKeys + (warp - 8) * 32 + lane + 32] = s1;
                }
                // dimensions 16 pc ...: pieces 2 (pc & 3), + 1 of panel pc / 4; the second panel's threads store the odd one first (banks)
                const int odd = pc >> 2;
                const uint32_t base = to + odd * kTcPanel + r0 * 128;
                const uint32_t c0 = base + (((2 * (pc & 3) + odd) ^ (r0 & 7)) << 4), c1 = base + (((2 * (pc & 3) + 1 - odd) ^ (r0 & 7)) << 4);
                uint4 raw[2][kRows];                               // (all on their way before the first is stored)
#pragma unroll
                for (int side = 0; side < 2; ++side)
#pragma unroll
                    for (int i = 0; i < kRows; ++i)                // rows r0 + 16 i: the same low bits
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[side][i].x), "=r"(raw[side][i].y), "=r"(raw[side][i].z), "=r"(raw[side][i].w)
                                     : "r"(from + place + side * kSideOff + i * kRowOff));
#pragma unroll
                for (int side = 0; side < 2; ++side)
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        const uint4 w = raw[side][i];
                        uint4 lo, hi;
                        codes_f16(odd ? w.z : w.x, lo.x, lo.y);
                        codes_f16(odd ? w.w : w.y, lo.z, lo.w);
                        codes_f16(odd ? w.x : w.z, hi.x, hi.y);
                        codes_f16(odd ? w.y : w.w, hi.z, hi.w);
                        const uint32_t at = side * 2 * kTcPanel + i * kRowOff;
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(c0 + at), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(c1 + at), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
                    }
                raw_out = raw_out == Sh::kRaws - 1 ? 0 : raw_out + 1;
            }
            fence_proxy_async();
            mbar_arrive(bar(Sh::kFullKV + st));
            ++it_out;
            if (++st_out == NS) {
                st_out = 0;
                lap_out ^= 1;
            }
            issue();
        }
        lm::cp_async_wait<0>();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sh::kRegsSoftmax));
        // ---- softmax, a thread per row of the stream's accumulator
        const int w = warp >> 2, rt = t & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + w * 256;
        // fp32: O of the tiles before, [four columns][row], relative to the maximum and scale that it had then
        float4* kept = kSplit ? reinterpret_cast<float4*>(a.kept) + ((size_t)c * 2 + w) * (kHd / 4) * 128 + rt : nullptr;
        int x = x_first, st = 0, kb = 0, nth = 0;
        uint32_t lap = 0;
        Part p;
        for (; next_part(x, p) && !*abort_flag; ++nth) {
            const int ctx = min(p.first, a.c.max_seq), r0 = (warp & 3) * 32;
            const int grow = p.group * a.group_rows + (kTall ? w * 128 : 0) + r0;      // the warp's first row, of the head's
            const int nn = min(32, p.nodes * a.group - grow);                          // and how many it has
            const bool active = nn > 0;
            // ---- the query rows, the largest element of each brought to 1 .. 2.  A warp copies its 32 rows, whole lines at a time, to where the
            // operand will lie (a row of bf16 takes the place of its f16, one of fp32 that of high parts and remainders); then a thread takes a
            // row.  kTall: each stream its own rows, else stream 0 those of both.
            float qf = 0.f;
            unsigned long long mask = 0;
            const bool mine = lane < nn;
            const uint32_t node = (uint32_t)(grow + lane) / (uint32_t)a.group;
            const size_t at_row = (((size_t)p.m * a.T + node) * a.nq + p.head * a.group + grow + lane - node * a.group) * kHd;
            if (!kTall && nth > 0) wait(Sh::kTaken, (nth - 1) & 1);   // O of both streams has been read
            if (mine) mask = mask_of(a, p.m, node, p.nodes) & low_bits((int)min((long)p.first + p.nodes, (long)a.c.max_seq) - ctx);
            constexpr int kLanes = kHd * (int)sizeof(A) / 16, kAtOnce = 32 / kLanes;       // 16-byte pieces of a row, rows at once
            const uint32_t tile = sq + (kTall ? w : 0) * (kSplit ? 2 : 1) * Sh::kQTile + r0 * 128;
            // piece j of the warp's row i: 1,024 bytes apart are rows 8 apart, 16 KB panels; within a row's 128 bytes swizzled
            auto place = [&](int i, int j) { return tile + (j >> 3) * 2 * kTcPanel + i * 128 + (((j & 7) ^ (i & 7)) << 4); };
            if (active && (kTall || w == 0)) {
                const int piece = lane % kLanes;
                int row = lane / kLanes, nd = (uint32_t)(grow + row) / (uint32_t)a.group, hd = grow + row - nd * a.group;
                const A* q = static_cast<const A*>(a.q) + (((size_t)p.m * a.T + nd) * a.nq + p.head * a.group + hd) * kHd + piece * (16 / (int)sizeof(A));
                const size_t skip = (size_t)(a.nq - a.group) * kHd;
#pragma unroll 4
                for (; row < nn; row += kAtOnce) {
                    amma::cp_async16(place(row, piece), q);
                    q += kAtOnce * kHd;
                    for (hd += kAtOnce; hd >= a.group; hd -= a.group) q += skip;
                }
                lm::cp_async_commit();
                lm::cp_async_wait<0>();
                __syncwarp();
                if (mine) {
                    uint4 raw[kLanes];
                    float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < kLanes; ++j) {
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[j].x), "=r"(raw[j].y), "=r"(raw[j].z), "=r"(raw[j].w) : "r"(place(lane, j)));
                        const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            mx[e] = kSplit ? fmaxf(mx[e], fabsf(__uint_as_float(u[e])))
                                           : fmaxf(fmaxf(mx[e], fabsf(__uint_as_float(u[e] << 16))), fabsf(__uint_as_float(u[e] & 0xFFFF0000u)));
                    }
                    const float2 unit = binade(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                    qf = unit.x * (0.08838834764831845f * 1.4426950408889634f);
#pragma unroll
                    for (int ch = 0; ch < 16; ++ch) {              // eight dimensions
                        float v[8];
                        if (kSplit) {
                            const uint4 x = raw[(2 * ch) % kLanes], y = raw[(2 * ch + 1) % kLanes];
                            v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
                            v[4] = __uint_as_float(y.x); v[5] = __uint_as_float(y.y); v[6] = __uint_as_float(y.z); v[7] = __uint_as_float(y.w);
                        } else {
                            const uint4 x = raw[ch % kLanes];
                            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                v[2 * e] = __uint_as_float(u[e] << 16);
                                v[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
                            }
                        }
                        uint32_t h[4], l[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            mul2(v[2 * e], v[2 * e + 1], unit.y, unit.y);
                            if (kSplit) {
                                amma::split_hi_lo(v[2 * e], v[2 * e + 1], h[e], l[e]);
                            } else {
                                const __half2 f = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
                                h[e] = *reinterpret_cast<const uint32_t*>(&f);
                            }
                        }
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, ch)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                        if (kSplit)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, ch) + Sh::kQTile), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
                    }
                }
                if (!kTall) s_qf[rt] = qf;
            }
            fence_proxy_async();
            mbar_arrive(bar(Sh::kFullQ));
            if (!kTall && w == 1) {
                wait(Sh::kFullQ, nth & 1);
                if (mine) qf = s_qf[rt];
            }
            float m = -FLT_MAX, l = 0.f, vunit = 1.f, m_kept = -FLT_MAX;
            bool has_kept = false;
            const int tiles = p.t1 - p.t0, jobs = kTall ? tiles : (tiles + 1 - w) >> 1;
            auto walk = [&]() {                               // a tile on in the ring of stages
                if (++st == NS) {
                    st = 0;
                    lap ^= 1;
                }
            };
            if (!kTall && w == 1) walk();
            for (int k = 0; k < jobs && !*abort_flag; ++k) {
                const int kk = kb + k, b = kk & 1, p0 = (p.t0 + (kTall ? k : 2 * k + w)) * kTcKeys;
                const uint32_t at = lanes + b * 64;
                wait(Sh::kFullS + 2 * w + b, (kk >> 1) & 1);
                if (kk > 1) wait(Sh::kDoneO + 2 * w + b, ((kk - 2) >> 1) & 1);   // long done; no phase of it goes by unseen
                if (kCoded) wait(Sh::kFullKV + st, lap);                         // (long full: the scales)
                tc::tc_fence_after();
                if (active) {
                    if (kSplit && k > 0 && k % kFlush == 0) {                    // O so far to the sum; the next product starts afresh
                        wait(Sh::kDoneO + 2 * w + (b ^ 1), ((kk - 1) >> 1) & 1);
                        tc::tc_fence_after();
                        const float f = has_kept ? lm::exp2_fast(m_kept - m) : 0.f;
#pragma unroll 1
                        for (int d = 0; d < kHd; d += 64) {                      // (half of it on its way at once: the latency of L2)
                            uint32_t o[64];
                            float4 old[16];
                            tc::tmem_ld32(lanes + 128 + d, o);
                            tc::tmem_ld32(lanes + 160 + d, o + 32);
#pragma unroll
                            for (int i = 0; i < 16; ++i) old[i] = has_kept ? kept[(d / 4 + i) * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                kept[(d / 4 + i) * 128] =
                                    make_float4(fmaf(old[i].x, f, __uint_as_float(o[4 * i])), fmaf(old[i].y, f, __uint_as_float(o[4 * i + 1])),
                                                fmaf(old[i].z, f, __uint_as_float(o[4 * i + 2])), fmaf(old[i].w, f, __uint_as_float(o[4 * i + 3])));
                        }
                        has_kept = true;
                        m_kept = m;
                    }
                    uint32_t r[64];
                    tc::tmem_ld32(at, r);
                    tc::tmem_ld32(at + 32, r + 32);
                    tc::tmem_wait_ld();
                    const float* ks = s_scale + st * 2 * kTcKeys;
                    const float* vs = ks + kTcKeys;
                    if (kCoded) {
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(ks + i);
                            mul2(r[i], r[i + 1], f.x, f.y);
                            mul2(r[i + 2], r[i + 3], f.z, f.w);
                        }
                    }
                    if (p0 + kTcKeys > ctx) {                                    // masks where the tile reaches the nodes
                        const unsigned long long vis = p0 >= ctx ? (p0 - ctx < 64 ? mask >> (p0 - ctx) : 0) : low_bits(ctx - p0) | mask << (ctx - p0);
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (!(vis >> i & 1)) r[i] = 0xFF800000u;
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; i += 8)
#pragma unroll
                        for (int d = 0; d < 4; ++d) mx[d] = fmaxf(fmaxf(mx[d], __uint_as_float(r[i + d])), __uint_as_float(r[i + 4 + d]));
                    float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * qf;
                    if (kCoded && k == 0) vunit = s_unit[st];
                    // Codes: the row's largest score beside the tile's largest value scale, a bound that is near enough where the scales are of one size.
                    const float bound = kCoded ? top + s_top[st] : top;
                    if (__any_sync(0xffffffffu, bound > m + kSlack)) {
                        top = bound;
                        if (kCoded && s_top[st] - s_low[st] > kNear) {
                            top = -INFINITY;
#pragma unroll
                            for (int i = 0; i < 64; i += 4) {
                                const float4 f = *reinterpret_cast<const float4*>(vs + i);
                                top = fmaxf(top, fmaxf(fmaxf(fmaf(__uint_as_float(r[i]), qf, scale_log2(f.x)), fmaf(__uint_as_float(r[i + 1]), qf, scale_log2(f.y))),
                                                       fmaxf(fmaf(__uint_as_float(r[i + 2]), qf, scale_log2(f.z)), fmaf(__uint_as_float(r[i + 3]), qf, scale_log2(f.w)))));
                            }
                        }
                        const float to = fmaxf(m, top - kHead);
                        const float2 h = step<kCoded>(m, to);
                        const float f = h.x * h.y;
                        const bool moves = !kCoded || __any_sync(0xffffffffu, to > m);
                        m = to;
                        l = l * h.x * h.y;
                        if (moves && (kSplit ? k % kFlush != 0 : k > 0)) {
                            wait(Sh::kDoneO + 2 * w + (b ^ 1), ((kk - 1) >> 1) & 1);   // O is complete up to the tile before
                            tc::tc_fence_after();
#pragma unroll 1
                            for (int d = 0; d < kHd; d += 16) {
                                uint32_t o[16];
                                tc::tmem_ld16(lanes + 128 + d, o);
                                tc::tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc::tmem_st16(lanes + 128 + d, o);
                            }
                        }
                    }
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i0 = 0; i0 < 64; i0 += kSplit ? 16 : 32) {  // P over the columns of 16 (fp32: then its remainders) or 32 positions
                        uint32_t h[16];
#pragma unroll
                        for (int i = 0; i < (kSplit ? 16 : 32); i += 4) {
                            float e[4];
#pragma unroll
                            for (int d = 0; d < 4; ++d) e[d] = __uint_as_float(r[i0 + i + d]);
                            fma2(e[0], e[1], qf, -m);
                            fma2(e[2], e[3], qf, -m);
#pragma unroll
                            for (int d = 0; d < 4; ++d) e[d] = lm::exp2_fast(e[d]);
                            add2(sum[0], sum[1], e[0], e[1]);
                            add2(sum[2], sum[3], e[2], e[3]);
                            if (kCoded) {
                                const float4 f = *reinterpret_cast<const float4*>(vs + i0 + i);
                                mul2(e[0], e[1], f.x, f.y);
                                mul2(e[2], e[3], f.z, f.w);
                            }
                            if (kSplit) {
                                split2(e[0], e[1], h[i / 2], h[(8 + i / 2) & 15]);
                                split2(e[2], e[3], h[i / 2 + 1], h[(9 + i / 2) & 15]);
                            } else {
                                const __half2 h0 = __floats2half2_rn(e[0], e[1]), h1 = __floats2half2_rn(e[2], e[3]);
                                h[i / 2] = *reinterpret_cast<const uint32_t*>(&h0);
                                h[i / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
                            }
                        }
                        tc::tmem_st16(at + i0, h);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc::tmem_wait_st();
                }
                tc::tc_fence_before();
                __syncwarp();
                mbar_arrive_by(lane == 0, bar(Sh::kFullP + 2 * w + b));
                walk();
                if (!kTall && (k + 1 < jobs || (w == 0 && tiles % 2 == 0))) walk();
            }
            if (!kTall && w == 1 && jobs > 0 && tiles % 2 == 1) walk();
            // ---- the part's end
            const int last = kb + jobs - 1;
            if (jobs > 0) wait(Sh::kDoneO + 2 * w + (last & 1), (last >> 1) & 1);
            tc::tc_fence_after();
            // kTall: a stream has its rows' results.  Otherwise both have a share of the same rows, O in the same lanes of tensor memory: with
            // the other's maximum, sum and scale, each joins half of the columns.
            float top = m, c0 = vunit, c1 = 0.f, f0 = has_kept ? lm::exp2_fast(m_kept - m) * vunit : 0.f, f1 = 0.f;
            const bool other = ((tiles + w) >> 1) > 0;               // the other stream had a tile
            if (!kTall) {
                s_ml[w * 128 + rt] = make_float4(m, l, c0, f0);
                mbar_arrive(bar(Sh::kGive));
                wait(Sh::kGive, nth & 1);
                tc::tc_fence_after();
                const float4 ml = s_ml[(w ^ 1) * 128 + rt];
                top = fmaxf(m, ml.x);
                const float2 h0 = step<kCoded>(m, top), h1 = step<kCoded>(ml.x, top);
                const float e0 = h0.x * h0.y, e1 = h1.x * h1.y;
                l = fmaf(l * h0.y, h0.x, ml.y * h1.x * h1.y);
                c0 *= e0;
                f0 *= e0;
                c1 = ml.z * e1;
                f1 = ml.w * e1;
            }
            if (active) {
                const bool whole = p.slot < 0;
                const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;   // (a row that sees nothing: 0)
                c0 *= inv; c1 *= inv; f0 *= inv; f1 *= inv;
                // A record is [four columns][row], then the rows' maxima and sums: a warp stores 512 bytes at once.
                float4* rec = whole ? nullptr : reinterpret_cast<float4*>(a.part + (size_t)p.slot * a.rec_rows * kPart) + (kTall ? w * 128 : 0) + rt;
                A* out = static_cast<A*>(a.out) + at_row;
                const float4* kept1 = kSplit ? reinterpret_cast<const float4*>(a.kept) + ((size_t)c * 2 + (w ^ 1)) * (kHd / 4) * 128 + rt : nullptr;
                constexpr int kCols = kTall && kSplit ? 64 : 16;              // columns on their way at once
#pragma unroll 1
                for (int d = kTall ? 0 : w * 64; d < (kTall ? kHd : w * 64 + 64); d += kCols) {
                    uint32_t o[kCols], q[kTall ? 16 : kCols];
                    float4 old[kSplit ? kCols / 4 : 1], old1[kSplit && !kTall ? kCols / 4 : 1];
#pragma unroll
                    for (int i = 0; i < kCols; i += 16) {
                        tc::tmem_ld16(lanes + 128 + d + i, reinterpret_cast<uint32_t(&)[16]>(o[i]));
                        if (!kTall) tc::tmem_ld16((lanes ^ 256) + 128 + d + i, reinterpret_cast<uint32_t(&)[16]>(q[kTall ? 0 : i]));
                    }
                    if (kSplit) {
#pragma unroll
                        for (int i = 0; i < kCols / 4; ++i) {
                            old[kSplit ? i : 0] = f0 != 0.f ? kept[(d / 4 + i) * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
                            if (!kTall) old1[kSplit && !kTall ? i : 0] = f1 != 0.f ? kept1[(d / 4 + i) * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                    }
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int i0 = 0; i0 < kCols; i0 += 16) {
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            v[i] = jobs > 0 ? __uint_as_float(o[i0 + i]) * c0 : 0.f;
                            if (!kTall && other) v[i] = fmaf(__uint_as_float(q[kTall ? 0 : i0 + i]), c1, v[i]);
                        }
                        if (kSplit) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const float4 x = old[kSplit ? (i0 + i) / 4 : 0], y = old1[kSplit && !kTall ? (i0 + i) / 4 : 0];
                                v[i] = fmaf(x.x, f0, v[i]); v[i + 1] = fmaf(x.y, f0, v[i + 1]); v[i + 2] = fmaf(x.z, f0, v[i + 2]); v[i + 3] = fmaf(x.w, f0, v[i + 3]);
                                if (!kTall) {
                                    v[i] = fmaf(y.x, f1, v[i]); v[i + 1] = fmaf(y.y, f1, v[i + 1]); v[i + 2] = fmaf(y.z, f1, v[i + 2]); v[i + 3] = fmaf(y.w, f1, v[i + 3]);
                                }
                            }
                        }
                        if (mine) {
                            if (!kTall && whole) {
                                store_o16(out + d + i0, v);
                            } else if (whole) {
                                // to where the query row lay: the stream's products are over
#pragma unroll
                                for (int i = 0; i < (kSplit ? 4 : 2); ++i) {
                                    const uint4 x = kSplit ? make_uint4(__float_as_uint(v[(4 * i) & 15]), __float_as_uint(v[(4 * i + 1) & 15]), __float_as_uint(v[(4 * i + 2) & 15]),
                                                                        __float_as_uint(v[(4 * i + 3) & 15]))
                                                           : make_uint4(lm::pack_bf16(v[(8 * i) & 15], v[(8 * i + 1) & 15]), lm::pack_bf16(v[(8 * i + 2) & 15], v[(8 * i + 3) & 15]),
                                                                        lm::pack_bf16(v[(8 * i + 4) & 15], v[(8 * i + 5) & 15]), lm::pack_bf16(v[(8 * i + 6) & 15], v[(8 * i + 7) & 15]));
                                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, (d + i0) * (int)sizeof(A) / 16 + i)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i += 4)
                                    rec[(size_t)((d + i0 + i) / 4) * a.rec_rows] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                            }
                        }
                    }
                }
                if (kTall && whole) {                                        // whole lines at a time from there (a row by a thread: 13 % more for short contexts)
                    __syncwarp();
                    const int piece = lane % kLanes;
                    int row = lane / kLanes, nd = (uint32_t)(grow + row) / (uint32_t)a.group, hd = grow + row - nd * a.group;
                    A* to = static_cast<A*>(a.out) + (((size_t)p.m * a.T + nd) * a.nq + p.head * a.group + hd) * kHd + piece * (16 / (int)sizeof(A));
                    const size_t skip = (size_t)(a.nq - a.group) * kHd;
#pragma unroll 4
                    for (; row < nn; row += kAtOnce) {
                        uint4 x;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(place(row, piece)) : "memory");
                        *reinterpret_cast<uint4*>(to) = x;
                        to += kAtOnce * kHd;
                        for (hd += kAtOnce; hd >= a.group; hd -= a.group) to += skip;
                    }
                    __syncwarp();                                            // (the next part's query rows come there)
                }
                if (!whole && mine && (kTall || w == 0)) {
                    *reinterpret_cast<float2*>(rec + (size_t)(kHd / 4) * a.rec_rows) = make_float2(top, l);
                }
            }
            if (!kTall) mbar_arrive(bar(Sh::kTaken));
            tc::tc_fence_before();
            kb += jobs;
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
    if (t == 0 && *abort_flag) atomicExch(a.status, kStatusMbarTimeout);
}

// Joins the records of contexts that several blocks have: a block per 32 rows and 64 columns of a head, a lane per row, eight columns per warp; from
// shared memory rows go out whole.
template <typename A>
__global__ void __launch_bounds__(256) attend_tc_merge_kernel(const Args a) {
    __shared__ __align__(16) float s_out[32][64 + 4];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = (blockIdx.x >> 1) * 32, c0 = (blockIdx.x & 1) * 64, head = blockIdx.y, m = blockIdx.z;
    const Seq q = seq_of(a, m);
    const int rows = q.nodes * a.group;
    if (q.tiles == 0 || r0 >= rows) return;
    const int g = r0 >= a.group_rows ? (uint32_t)r0 / (uint32_t)a.group_rows : 0, row = min(r0 + lane, rows - 1);
    const int x0 = a.cum[m] + (head * q.groups + g) * q.tiles, x1 = x0 + q.tiles;
    const int* starts = a.cum + kPlanned;                          // of the blocks' stretches, in tiles
    const float per = (float)a.blocks / (float)starts[a.blocks];
    auto block_of = [&](int x) {                                   // the block that has tile x
        int c = max(0, min((int)((float)x * per), a.blocks - 1));
        while (starts[c + 1] <= x) ++c;
        while (starts[c] > x) --c;
        return c;
    };
    const int b0 = block_of(x0), b1 = block_of(x1 - 1);
    if (b0 == b1) return;                                          // one block had it whole
    const size_t record = (size_t)a.rec_rows * (kPart / 4);
    const float4* rec = reinterpret_cast<const float4*>(a.part) + row - g * a.group_rows;
    const size_t late = starts[b0] < x0 ? record : 0;              // (the first block may have other work before)
    float top = -FLT_MAX, sum = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int b = b0; b <= b1; b += 4) {                            // four records in flight
        float v[4][8], mt[4], lt[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = min(b + j, b1);
            const bool there = b + j <= b1 && starts[c] < starts[c + 1];
            const float4* at = rec + 2 * c * record + (c == b0 ? late : 0);
            const float2 ml = there ? *reinterpret_cast<const float2*>(at + (size_t)(kHd / 4) * a.rec_rows) : make_float2(-FLT_MAX, 0.f);
            mt[j] = ml.x;
            lt[j] = ml.y;
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 x = there ? at[(size_t)((c0 + warp * 8 + i) / 4) * a.rec_rows] : make_float4(0.f, 0.f, 0.f, 0.f);
                v[j][i] = x.x; v[j][i + 1] = x.y; v[j][i + 2] = x.z; v[j][i + 3] = x.w;
            }
        }
        const float to = fmaxf(top, fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3])));
        const float2 h = step<true>(top, to);
        const float f = h.x * h.y;
        top = to;
        sum = sum * h.x * h.y;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 h = step<true>(mt[j], to);
            const float e = h.x * h.y;
            sum = fmaf(lt[j] * h.y, h.x, sum);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(v[j][i], e, acc[i]);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 8; i += 4)
        *reinterpret_cast<float4*>(&s_out[lane][warp * 8 + i]) = make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = r0 + 2 * warp + (lane >> 4) + 16 * i;
        if (r >= rows) break;
        const uint32_t node = (uint32_t)r / (uint32_t)a.group;
        lm::store4(static_cast<A*>(a.out) + (((size_t)m * a.T + node) * a.nq + head * a.group + r - node * a.group) * kHd + c0 + 4 * (lane & 15),
                 *reinterpret_cast<const float4*>(&s_out[r - r0][4 * (lane & 15)]));
    }
}

}  // namespace tree
}  // namespace bw
