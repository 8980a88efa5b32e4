// The same attention on the 5th-generation tensor cores.
//
// One block of 512 threads per SM.  Query rows (node, query head of the group) are the 128 lanes of an accumulator; two accumulator sets
// ("streams") keep the tensor cores busy while the softmax of one runs:
//   kTall   more than 128 rows: each stream has 128 rows, both take every 64 positions of the context
//   else    each stream has all rows and takes every other 64 positions; stream 1 hands its result to stream 0 at the end
// Warps 0-3 and 4-7: softmax of a stream, a thread per row.  Warps 8-11: the cache; binary16 rows go to their swizzled place by cp.async, codes
// come raw, become f16 (exact) and are stored there.  Warp 12 issues the products:
//   S = Q K^T    two S buffers of 64 columns per stream, the next scores are on their way while the softmax has these
//   O += P V     P over the scores' columns as the f16 A operand, V from shared memory as it lies there ([position][column])
// fp32 activations: Q and P as f16 high parts and remainders, multiplied one after the other.  The accumulator's sums are cut, not rounded, at
// 24 bits, which adds up over a long context: there O is taken to registers every eight tiles and starts afresh.
// Scales and the moving maximum as in attention_tree.cuh; a warp brings its rows of O to a new maximum by itself.
// Work is shared out in tiles of 64 positions: all sequences' tiles, heads and row groups in one line, an equal stretch of it per block; what
// a block has of a head's context that it does not have whole goes to a record that the merge kernel joins.
// All waits are bounded; a wait that gives up raises an abort flag.
#pragma once
#include "attention_tree.cuh"
#include "gemm_w4a8_tc.cuh"

namespace bw {
namespace tree {

constexpr int kTcKeys = 64, kTcPanel = kTcKeys * 128, kTcThreads = 512;   // positions of a tile, bytes of 64 x 64 f16
constexpr int kTcStage = 4 * kTcPanel;                                    // K and V of a tile
constexpr int kTcRaw = 2 * kTcKeys * kHd + 2 * kTcKeys * 4;               // codes and scales of a tile
constexpr int kFlush = 8;
constexpr int kPlanned = 512;                                              // sequences whose work is laid out in a line

template <bool kTall, bool kCoded, bool kSplit>
struct TcShape {
    static constexpr int kQTile = 4 * kTcPanel;                                      // 128 rows x 128
    static constexpr int kQ = (kTall ? 2 : 1) * (kSplit || !kTall ? 2 : 1) * kQTile; // (64 KB at least where it serves the hand-over too)
    static constexpr int kStages = kTall && kSplit ? 2 : kCoded ? 3 : 4;
    static constexpr int kRaws = !kCoded ? 0 : kTall && kSplit ? 1 : 3;
    static constexpr int kHead = 4096;                                               // barriers, the line of work, what stream 1 hands over
    static constexpr int kScales = (kStages * 2 * kTcKeys * 4 + 1023) / 1024 * 1024;
    static constexpr int kSmem = 1024 + kHead + kScales + kQ + kStages * kTcStage + kRaws * kTcRaw;
    static_assert(kSmem <= 232448, "shared memory of a block");
    // registers per thread: 256 softmax threads, 256 others; 65,536 together, what 512 threads of 128 start with
    static constexpr int kRegsSoftmax = kSplit ? 208 : 152, kRegsOther = 256 - kRegsSoftmax;
    static constexpr int kPiece = kSplit ? 16 : 32;                                  // columns of scores that a thread holds at once
    // barriers
    static constexpr int kFullQ = 0, kFullS = 1, kFullP = 5, kDoneO = 9, kDrain = 13, kGive = 14, kGiven = 15, kTaken = 16, kFullKV = 17,
                         kEmptyKV = kFullKV + kStages, kBars = kEmptyKV + kStages;
};

// ------------------------------------------------------------------------------------------------------------------ work in a line
struct Part {
    int m, head, group, t0, t1, slot;   // slot < 0: the head's whole context
};
__device__ __forceinline__ int seq_end(const Args& a, int m, int nodes) { return (int)min((long)a.first[m] + nodes, (long)a.c.max_seq); }
__device__ __forceinline__ int seq_tiles(const Args& a, int m, int* groups) {
    const int nodes = node_count(a, m);
    *groups = (nodes * a.group + a.group_rows - 1) / a.group_rows;
    if (a.first[m] < 0 || nodes == 0) { *groups = 0; return 0; }
    return (seq_end(a, m, nodes) + kTcKeys - 1) / kTcKeys;
}

template <bool kTall, bool kCoded, typename A>
__global__ void __launch_bounds__(kTcThreads, 1) attend_tc_kernel(const Args a) {
    constexpr bool kSplit = sizeof(A) == 4;
    using Sh = TcShape<kTall, kCoded, kSplit>;
    constexpr int NS = Sh::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_area = smem + Sh::kHead + Sh::kScales;       // (a multiple of 1,024 from the base)
    static_assert((Sh::kHead + Sh::kScales) % 1024 == 0, "swizzled tiles start at 1,024 bytes");
    const uint32_t sq = smem_u32(q_area), skv = sq + Sh::kQ, sraw = skv + NS * kTcStage, bar0 = smem_u32(smem), flag = bar0 + 516;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 516);
    int* s_cum = reinterpret_cast<int*>(smem + 768);               // [kPlanned + 1]
    float2* s_ml = reinterpret_cast<float2*>(smem + 3072);         // [128]
    float* s_scale = reinterpret_cast<float*>(smem + Sh::kHead);   // [stage][K 64, V 64]
    float* s_vtop = reinterpret_cast<float*>(smem + 520);          // [stage][2]
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
        mbar_init(bar(Sh::kDrain), 1);
        mbar_init(bar(Sh::kGive), 128);
        mbar_init(bar(Sh::kGiven), 128);
        mbar_init(bar(Sh::kTaken), 128);
        for (int i = 0; i < NS; ++i) {
            mbar_init(bar(Sh::kFullKV + i), 128);
            mbar_init(bar(Sh::kEmptyKV + i), 1);
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
        int groups, v = 0;
        if (t < a.M) {
            v = seq_tiles(a, t, &groups);
            v *= groups * a.c.heads;
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
        for (int w = 0; w < 16; ++w) {
            before += w < warp ? s_warp[w] : 0;
            line += s_warp[w];
        }
        if (t < a.M) s_cum[t] = before + sum - v;
        if (t == 0) s_cum[a.M] = line;
        if (blockIdx.x == 0) {                                     // for the merge
            if (t < a.M) a.cum[t] = before + sum - v;
            if (t <= a.blocks) a.cum[kPlanned + t] = (int)((long)line * t / a.blocks);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(smem + 512), 0);
    const int c = blockIdx.x, x_first = a.flat ? (int)((long)line * c / gridDim.x) : 0, x_end = a.flat ? (int)((long)line * (c + 1) / gridDim.x) : 1;
    // Part number 0, 1, ... of this block: false after the last.  x: where it starts in the line, moved on.
    auto next_part = [&](int& x, Part& p) {
        if (x >= x_end) return false;
        if (a.flat) {
            int lo = 0, hi = a.M - 1;                              // the last sequence that starts at or before x
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_cum[mid] <= x) lo = mid; else hi = mid - 1;
            }
            p.m = lo;
            int groups;
            const int tiles = seq_tiles(a, p.m, &groups), rel = x - s_cum[lo], pair = rel / tiles;
            p.head = pair / groups;
            p.group = pair - p.head * groups;
            p.t0 = rel - pair * tiles;
            p.t1 = min(tiles, p.t0 + x_end - x);
            p.slot = p.t0 == 0 && p.t1 == tiles ? -1 : 2 * c + (x == x_first ? 0 : 1);
            x += p.t1 - p.t0;
            return true;
        }
        x = 1;
        int groups;
        p.group = blockIdx.x % a.groups;
        p.head = blockIdx.x / a.groups % a.c.heads;
        p.m = blockIdx.x / a.groups / a.c.heads;
        p.t0 = 0;
        p.t1 = seq_tiles(a, p.m, &groups);
        p.slot = -1;
        return p.group < groups;
    };
    // Jobs of a part: job n is tile n / 2 (kTall) or n and stream n & 1; job k of stream w is n = 2 k + w.
    auto jobs_of = [&](const Part& p) { return (p.t1 - p.t0) * (kTall ? 2 : 1); };

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::kRegsOther));
        if (warp == 12) {
            // The whole warp walks the loop, one elected lane issues.
            constexpr uint32_t id_s = tc::idesc_f16(kTcKeys), id_o = tc::idesc_f16(kHd, true);
            const bool elected = tc::elect_one();
            int x = x_first, it0 = 0, kb[2] = {0, 0}, nth = 0;
            Part p;
            for (; next_part(x, p) && !*abort_flag; ++nth) {
                const int jobs = jobs_of(p);
                auto scores = [&](int n) {
                    const int w = n & 1, kk = kb[w] + (n >> 1), b = kk & 1, it = it0 + (kTall ? n >> 1 : n), st = it % NS;
                    if (kk > 1) wait(Sh::kDoneO + 2 * w + b, ((kk - 2) >> 1) & 1);   // the P that lay there has been multiplied
                    wait(Sh::kFullKV + st, (it / NS) & 1);
                    tc::tc_fence_after();
                    if (elected) {
                        const uint32_t d = tmem + w * 256 + b * 64, q = sq + (kTall ? w : 0) * (kSplit ? 2 : 1) * Sh::kQTile, k = skv + st * kTcStage;
#pragma unroll
                        for (int part = 0; part < (kSplit ? 2 : 1); ++part)
#pragma unroll
                            for (int pan = 0; pan < 2; ++pan)
#pragma unroll
                                for (int e = 0; e < 4; ++e)   // 16 dimensions = 32 bytes further inside the swizzle atom
                                    tc::tc_mma_bf16(d, tc::flash_desc(q + part * Sh::kQTile + pan * 2 * kTcPanel, 16, 1024) + 2 * e,
                                                    tc::flash_desc(k + pan * kTcPanel, 16, 1024) + 2 * e, id_s, part + pan + e > 0 ? 1u : 0u);
                        tc::tc_commit(bar(Sh::kFullS + 2 * w + b));
                    }
                    __syncwarp();
                };
                wait(Sh::kFullQ, nth & 1);
                tc::tc_fence_after();
                scores(0);
                if (jobs > 1) scores(1);
                for (int n = 0; n < jobs && !*abort_flag; ++n) {
                    if (n + 2 < jobs) scores(n + 2);
                    const int w = n & 1, k = n >> 1, kk = kb[w] + k, b = kk & 1, it = it0 + (kTall ? n >> 1 : n), st = it % NS;
                    wait(Sh::kFullP + 2 * w + b, (kk >> 1) & 1);
                    tc::tc_fence_after();
                    if (elected) {
                        const uint32_t pa = tmem + w * 256 + b * 64, o = tmem + w * 256 + 128, v = skv + st * kTcStage + 2 * kTcPanel;
                        const bool fresh = kSplit ? k % kFlush == 0 : k == 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {   // 16 positions: two 8-row groups
                            const uint64_t vd = tc::flash_desc(v, kTcPanel, 1024) + e * (2048 >> 4);
                            const uint32_t at = pa + (kSplit ? 16 * e : (e >> 1) * 32 + (e & 1) * 8);
                            tc::tc_mma_bf16_ta(o, at, vd, id_o, fresh && e == 0 ? 0u : 1u);
                            if (kSplit) tc::tc_mma_bf16_ta(o, at + 8, vd, id_o, 1u);
                        }
                        tc::tc_commit(bar(Sh::kDoneO + 2 * w + b));
                        if (!kTall || w == 1) tc::tc_commit(bar(Sh::kEmptyKV + st));
                    }
                    __syncwarp();
                }
                it0 += p.t1 - p.t0;
                kb[0] += (jobs + 1) >> 1;
                kb[1] += jobs >> 1;
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
        int xi = x_first, xo = x_first, it_in = 0, it_out = 0;
        Part in{}, out{};
        int in_tile = 0, out_tile = 0;
        bool in_more = next_part(xi, in), out_more = next_part(xo, out);
        in_tile = in.t0;
        out_tile = out.t0;
        int ctx = 0, end = 0;
        unsigned long long any = 0;
        const unsigned char *kp = nullptr, *vp = nullptr;
        size_t row0 = 0;
        auto open_part = [&]() {                                   // what the sequence's rows see
            const int nodes = node_count(a, in.m);
            ctx = min(a.first[in.m], a.c.max_seq);
            end = seq_end(a, in.m, nodes);
            const unsigned long long mine = (lane < nodes ? mask_of(a, in.m, lane, nodes) : 0) | (lane + 32 < nodes ? mask_of(a, in.m, lane + 32, nodes) : 0);
            any = (unsigned long long)__reduce_or_sync(0xffffffffu, (uint32_t)(mine >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)mine);
            row0 = a.c.row(in.m, in.head, 0);
            kp = a.c.k + row0 * kRowBytes;
            vp = a.c.v + row0 * kRowBytes;
        };
        auto issue = [&]() {                                       // the next tile on its way
            if (in_more) {
                if (in_tile == in.t0) open_part();
                const int p0 = in_tile * kTcKeys;
                const bool all = p0 + kTcKeys <= ctx;
                if (!kCoded) wait(Sh::kEmptyKV + it_in % NS, (it_in / NS & 1) ^ 1);
                const uint32_t to = kCoded ? sraw + it_in % max(Sh::kRaws, 1) * kTcRaw : skv + it_in % NS * kTcStage;
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const int r = r0 + kStep * i, p = p0 + r;
                    const bool there = all || p < ctx || (p < end && (any >> (p - ctx) & 1));
                    const size_t from = (size_t)(there ? p : 0) * kRowBytes + pc * 16;
                    if (kCoded) {
                        lm::cp_async16z(to + r * kHd + pc * 16, kp + from, there);
                        lm::cp_async16z(to + kTcKeys * kHd + r * kHd + pc * 16, vp + from, there);
                    } else {
                        const uint32_t at = to + (pc >> 3) * kTcPanel + r * 128 + (((pc & 7) ^ (r & 7)) << 4);
                        lm::cp_async16z(at, kp + from, there);
                        lm::cp_async16z(at + 2 * kTcPanel, vp + from, there);
                    }
                }
                if (kCoded) {
                    const int p = p0 + (u & 63);
                    const bool there = all || p < ctx || (p < end && (any >> (p - ctx) & 1));
                    tc::cp_async4(to + 2 * kTcKeys * kHd + u * 4, (u < 64 ? a.c.ks : a.c.vs) + row0 + (there ? p : 0), there ? 4 : 0);
                }
                ++it_in;
                if (++in_tile == in.t1) {
                    in_more = next_part(xi, in);
                    in_tile = in.t0;
                }
            }
            lm::cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) issue();
        while (out_more && !*abort_flag) {
            const int st = it_out % NS;
            lm::cp_async_wait<kAhead - 1>();
            if (kCoded) {
                wait(Sh::kEmptyKV + st, (it_out / NS & 1) ^ 1);
                const uint32_t from = sraw + it_out % max(Sh::kRaws, 1) * kTcRaw, to = skv + st * kTcStage;
                const float* fs = reinterpret_cast<const float*>(smem + (from - bar0) + 2 * kTcKeys * kHd);
                const float sc = fs[u];
                s_scale[st * 2 * kTcKeys + u] = sc;
                if (warp >= 10) {
                    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(sc)));
                    if (lane == 0) s_vtop[2 * st + warp - 10] = __uint_as_float(top);
                }
#pragma unroll
                for (int side = 0; side < 2; ++side)
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        const int r = r0 + kStep * i;
                        uint4 w;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                     : "r"(from + side * kTcKeys * kHd + r * kHd + pc * 16));
                        uint4 lo = make_uint4(codes_f16x2(w.x), codes_f16x2(w.x >> 16), codes_f16x2(w.y), codes_f16x2(w.y >> 16));
                        uint4 hi = make_uint4(codes_f16x2(w.z), codes_f16x2(w.z >> 16), codes_f16x2(w.w), codes_f16x2(w.w >> 16));
                        // dimensions 16 pc ...: pieces 2 (pc & 3), + 1 of panel pc / 4; the second panel's threads store the odd one first (banks)
                        const uint32_t base = to + side * 2 * kTcPanel + (pc >> 2) * kTcPanel + r * 128;
                        const int odd = pc >> 2;
                        const uint32_t c0 = base + (((2 * (pc & 3) + odd) ^ (r & 7)) << 4), c1 = base + (((2 * (pc & 3) + 1 - odd) ^ (r & 7)) << 4);
                        const uint4 first = odd ? hi : lo, second = odd ? lo : hi;
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(c0), "r"(first.x), "r"(first.y), "r"(first.z), "r"(first.w) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(c1), "r"(second.x), "r"(second.y), "r"(second.z), "r"(second.w) : "memory");
                    }
            }
            fence_proxy_async();
            mbar_arrive(bar(Sh::kFullKV + st));
            ++it_out;
            if (++out_tile == out.t1) {
                out_more = next_part(xo, out);
                out_tile = out.t0;
            }
            issue();
        }
        lm::cp_async_wait<0>();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sh::kRegsSoftmax));
        // ---- softmax, a thread per row of the stream's accumulator
        const int w = warp >> 2, rt = t & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + w * 256;
        int x = x_first, it0 = 0, kb = 0, nth = 0;
        Part p;
        for (; next_part(x, p) && !*abort_flag; ++nth) {
            const int nodes = node_count(a, p.m), ctx = min(a.first[p.m], a.c.max_seq);
            const int rows = nodes * a.group - p.group * a.group_rows - (kTall ? w * 128 : 0);   // of this stream, from its first lane on
            const bool active = (warp & 3) * 32 < rows, mine = rt < rows;
            const int row = p.group * a.group_rows + (kTall ? w * 128 : 0) + rt, node = mine ? row / a.group : 0;
            const unsigned long long mask = mine ? mask_of(a, p.m, node, nodes) & low_bits(seq_end(a, p.m, nodes) - ctx) : 0;
            // ---- the warp's query rows, the largest element of each brought to 1 .. 2: a row at a time, four dimensions a lane.  kTall: the
            // stream's own rows, else panel w of the rows that both streams have.
            float qf = 0.f;
            if (!kTall && nth > 0) wait(Sh::kTaken, (nth - 1) & 1);   // all rows of the hand-over have been read
            if (active) {
                const uint32_t tile = sq + (kTall ? w : 0) * (kSplit ? 2 : 1) * Sh::kQTile + (lane >> 4) * 2 * kTcPanel + (lane & 1) * 8;
                const int r0 = (warp & 3) * 32, grow = p.group * a.group_rows + (kTall ? w * 128 : 0) + r0;
                const A* q = static_cast<const A*>(a.q) + ((size_t)p.m * a.T * a.nq + p.head * a.group) * kHd + 4 * lane;
                const int nn = min(32, rows - r0);
                int nd = grow / a.group, hd = grow - nd * a.group;        // node and head of row i, walked along
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += 8) {
                    float4 v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[i] = i0 + i < nn ? load_q4(q + ((size_t)nd * a.nq + hd) * kHd) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (++hd == a.group) { hd = 0; ++nd; }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float top = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
                        const float2 unit = binade(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
                        if (lane == i0 + i) qf = unit.x * (0.08838834764831845f * 1.4426950408889634f);
                        uint32_t h[2], l[2];
                        amma::split_hi_lo(v[i].x * unit.y, v[i].y * unit.y, h[0], l[0]);
                        amma::split_hi_lo(v[i].z * unit.y, v[i].w * unit.y, h[1], l[1]);
                        const int r = r0 + i0 + i;
                        const uint32_t to = tile + r * 128 + (((lane >> 1 & 7) ^ (r & 7)) << 4);
                        if (kTall || lane >> 4 == w) {
                            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(h[0]), "r"(h[1]) : "memory");
                            if (kSplit) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + Sh::kQTile), "r"(l[0]), "r"(l[1]) : "memory");
                        }
                    }
                }
            }
            fence_proxy_async();
            mbar_arrive(bar(Sh::kFullQ));
            float m = -FLT_MAX, l = 0.f, vref = __uint_as_float(2u << 23);
            float kept[kSplit ? kHd : 1];
            if (kSplit) {
#pragma unroll
                for (int i = 0; i < (kSplit ? kHd : 1); ++i) kept[i] = 0.f;
            }
            const int jobs = (jobs_of(p) + 1 - w) >> 1;
            for (int k = 0; k < jobs && !*abort_flag; ++k) {
                const int kk = kb + k, b = kk & 1, rel = kTall ? k : 2 * k + w, it = it0 + rel, st = it % NS, p0 = (p.t0 + rel) * kTcKeys;
                const uint32_t at = lanes + b * 64;
                wait(Sh::kFullS + 2 * w + b, (kk >> 1) & 1);
                if (kk > 1) wait(Sh::kDoneO + 2 * w + b, ((kk - 2) >> 1) & 1);   // long done; no phase of it goes by unseen
                if (kCoded) wait(Sh::kFullKV + st, (it / NS) & 1);               // (long full: the scales)
                tc::tc_fence_after();
                if (kSplit && k > 0 && k % kFlush == 0 && active) {             // O so far to registers; the next product starts afresh
                    wait(Sh::kDoneO + 2 * w + (b ^ 1), ((kk - 1) >> 1) & 1);
                    tc::tc_fence_after();
#pragma unroll
                    for (int d = 0; d < (kSplit ? kHd : 0); d += 32) {
                        uint32_t o[32];
                        tc::tmem_ld32(lanes + 128 + d, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) kept[d + i] += __uint_as_float(o[i]);
                    }
                }
                if (active) {
                    const float* ks = s_scale + st * 2 * kTcKeys;
                    const float* vs = ks + kTcKeys;
                    const bool tail = p0 + kTcKeys > ctx;
                    unsigned long long vis = ~0ull;
                    if (tail) vis = p0 >= ctx ? (p0 - ctx < 64 ? mask >> (p0 - ctx) : 0) : low_bits(ctx - p0) | mask << (ctx - p0);
                    constexpr int kPiece = Sh::kPiece;
                    auto scores = [&](int i0, float (&s)[kPiece]) {      // of positions i0 ..., times the keys' scales
                        uint32_t r[kPiece];
                        if constexpr (kPiece == 32) tc::tmem_ld32(at + i0, r);
                        else tc::tmem_ld16(at + i0, r);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < kPiece; i += 4) {
                            float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
                            if (kCoded) f = *reinterpret_cast<const float4*>(ks + i0 + i);
                            s[i] = __uint_as_float(r[i]); s[i + 1] = __uint_as_float(r[i + 1]);
                            s[i + 2] = __uint_as_float(r[i + 2]); s[i + 3] = __uint_as_float(r[i + 3]);
                            if (kCoded) { s[i] *= f.x; s[i + 1] *= f.y; s[i + 2] *= f.z; s[i + 3] *= f.w; }
                        }
                        if (tail) {
                            const uint32_t bits = (uint32_t)(vis >> i0);
#pragma unroll
                            for (int i = 0; i < kPiece; ++i)
                                if (!(bits >> i & 1)) s[i] = -INFINITY;
                        }
                    };
                    float s[kPiece], mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i0 = 0; i0 < kTcKeys; i0 += kPiece) {
                        scores(i0, s);
#pragma unroll
                        for (int i = 0; i < kPiece; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                    }
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * qf;
                    float vtop = vref;
                    if (kCoded) vtop = fmaxf(s_vtop[2 * st], s_vtop[2 * st + 1]);
                    if (__any_sync(0xffffffffu, top > m + kSlack || vtop > vref)) {
                        float f = 1.f;
                        if (kCoded && vtop > vref) {
                            const float to = __uint_as_float(min((__float_as_uint(vtop) + 0x7FFFFFu) & 0x7F800000u, 252u << 23));
                            f = vref * __uint_as_float((254u << 23) - __float_as_uint(to));
                            vref = to;
                        }
                        const float to = fmaxf(m, top - kHead), e = lm::exp2_fast(m - to);
                        m = to;
                        l *= e;
                        f *= e;
                        if (kSplit) {
#pragma unroll
                            for (int i = 0; i < (kSplit ? kHd : 1); ++i) kept[i] *= f;
                        }
                        if (kSplit ? k % kFlush != 0 : k > 0) {
                            wait(Sh::kDoneO + 2 * w + (b ^ 1), ((kk - 1) >> 1) & 1);   // O is complete up to the tile before
                            tc::tc_fence_after();
#pragma unroll
                            for (int d = 0; d < kHd; d += 32) {
                                uint32_t o[32];
                                tc::tmem_ld32(lanes + 128 + d, o);
                                tc::tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc::tmem_st32(lanes + 128 + d, o);
                            }
                        }
                    }
                    const float vdiv = kCoded ? __uint_as_float((254u << 23) - __float_as_uint(vref)) : 1.f;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i0 = 0; i0 < kTcKeys; i0 += kPiece) {       // P over the same columns, 16 of them: high parts, then (fp32) remainders
                        scores(i0, s);
                        uint32_t h[16];
#pragma unroll
                        for (int i = 0; i < kPiece; i += 4) {
                            float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
                            if (kCoded) f = *reinterpret_cast<const float4*>(vs + i0 + i);
                            float e[4];
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                e[d] = lm::exp2_fast(fmaf(s[i + d], qf, -m));
                                sum[d] += e[d];
                            }
                            if (kCoded) { e[0] *= f.x * vdiv; e[1] *= f.y * vdiv; e[2] *= f.z * vdiv; e[3] *= f.w * vdiv; }
                            if (kSplit) {
                                amma::split_hi_lo(e[0], e[1], h[i / 2], h[(8 + i / 2) & 15]);
                                amma::split_hi_lo(e[2], e[3], h[i / 2 + 1], h[(9 + i / 2) & 15]);
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
            }
            // ---- the part's end
            const int last = kb + jobs - 1;
            if (jobs > 0) wait(Sh::kDoneO + 2 * w + (last & 1), (last >> 1) & 1);
            tc::tc_fence_after();
            // Each warp's 16 KB of the queries' place: what stream 1 has, [column][row]; then, 32 columns at a time, [row][column] with the
            // 16-byte pieces swizzled, from where rows go out whole lines at a time.
            float* hand = reinterpret_cast<float*>(q_area + (kTall ? w * (kSplit ? 2 : 1) * Sh::kQTile + (warp & 3) * 4096 : (warp & 3) * 16384));
            float top = m, c0 = 1.f, c1 = 0.f;
            if (!kTall) {
                if (w == 0) {
                    mbar_arrive(bar(Sh::kGive));              // both streams' scores are done: the queries' place is free
                    wait(Sh::kGiven, nth & 1);
                    const float2 ml = s_ml[rt];
                    top = fmaxf(m, ml.x);
                    c0 = lm::exp2_fast(m - top);
                    c1 = lm::exp2_fast(ml.x - top);
                    l = fmaf(l, c0, ml.y * c1);
                } else {
                    wait(Sh::kGive, nth & 1);
                    s_ml[rt] = make_float2(m, l);
                }
            }
            if (active) {
                const float vmul = kCoded ? vref : 1.f, inv = l == 0.f ? 0.f : 1.f / l;
                const bool whole = p.slot < 0;
                const int r0 = (warp & 3) * 32, nn = min(32, rows - r0), grow = p.group * a.group_rows + (kTall ? w * 128 : 0) + r0;
                float* rec = whole ? nullptr : a.part + ((size_t)p.slot * a.rec_rows + (kTall ? w * 128 : 0) + r0) * kPart;
                A* out = static_cast<A*>(a.out) + ((size_t)p.m * a.T * a.nq + p.head * a.group) * kHd;
#pragma unroll
                for (int d = 0; d < kHd; d += 32) {
                    uint32_t o[32];
                    if (jobs > 0) {
                        tc::tmem_ld32(lanes + 128 + d, o);
                        tc::tmem_wait_ld();
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float v = jobs > 0 ? __uint_as_float(o[i]) : 0.f;
                        if (kSplit) v += kept[kSplit ? d + i : 0];
                        v *= vmul;
                        if (!kTall && w == 1) hand[(d + i) * 32 + lane] = v;
                        if (!kTall && w == 0) v = fmaf(v, c0, c1 * hand[(d + i) * 32 + lane]);
                        o[i] = __float_as_uint(whole ? v * inv : v);
                    }
                    if (!kTall && w == 1) continue;
                    float* stage = hand + (kTall ? 0 : d * 32);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(stage + lane * 32 + ((i ^ (lane & 7)) << 2)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    __syncwarp();
#pragma unroll 2
                    for (int i = lane >> 3; i < nn; i += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(stage + i * 32 + (((lane & 7) ^ (i & 7)) << 2));
                        if (whole) {
                            const int nd = (grow + i) / a.group;
                            store_o4(out + ((size_t)nd * a.nq + grow + i - nd * a.group) * kHd + d + 4 * (lane & 7), v);
                        } else {
                            *reinterpret_cast<float4*>(rec + (size_t)i * kPart + d + 4 * (lane & 7)) = v;
                        }
                    }
                }
                if (!whole && mine && (kTall || w == 0)) *reinterpret_cast<float2*>(rec + (size_t)lane * kPart + kHd) = make_float2(top, l);
            }
            if (!kTall) mbar_arrive(bar(w == 1 ? Sh::kGiven : Sh::kTaken));
            tc::tc_fence_before();
            it0 += p.t1 - p.t0;
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

// Joins the records of contexts that several blocks have, a warp per row.
template <typename A>
__global__ void __launch_bounds__(128) attend_tc_merge_kernel(const Args a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 5);     // (m, head, row)
    if (at >= (long)a.M * a.c.heads * a.rows) return;
    const int row = (int)(at % a.rows), mh = (int)(at / a.rows), m = mh / a.c.heads, head = mh - m * a.c.heads, node = row / a.group;
    if (a.first[m] < 0 || node >= node_count(a, m)) return;
    int groups;
    const int tiles = seq_tiles(a, m, &groups), g = row / a.group_rows;
    const int x0 = a.cum[m] + (head * groups + g) * tiles, x1 = x0 + tiles;
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
    const bool late = starts[b0] < x0;                             // the first block has other work before
    auto record = [&](int c) { return a.part + ((size_t)(2 * c + (c == b0 && late ? 1 : 0)) * a.rec_rows + row - g * a.group_rows) * kPart; };
    float top = -FLT_MAX, sum = 0.f;
    for (int c = b0 + lane; c <= b1; c += 32)
        if (starts[c] < starts[c + 1]) top = fmaxf(top, record(c)[kHd]);
    top = warp_max(top);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = b0; c <= b1; ++c) {
        if (starts[c] == starts[c + 1]) continue;
        const float* rec = record(c);
        const float2 ml = *reinterpret_cast<const float2*>(rec + kHd);
        const float4 v = *reinterpret_cast<const float4*>(rec + 4 * lane);
        const float e = lm::exp2_fast(ml.x - top);
        sum = fmaf(ml.y, e, sum);
        acc.x = fmaf(v.x, e, acc.x); acc.y = fmaf(v.y, e, acc.y); acc.z = fmaf(v.z, e, acc.z); acc.w = fmaf(v.w, e, acc.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    A* out = static_cast<A*>(a.out) + (((size_t)m * a.T + node) * a.nq + head * a.group + row - node * a.group) * kHd + 4 * lane;
    store_o4(out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

}  // namespace tree
}  // namespace bw
