// Attention of single tokens and of drafted trees over a binary16 or 8-bit cache (attention_tree.cuh): splits and entry points.
#include "attention_tree_tc.cuh"

#include <mutex>

#include "host_util.h"

namespace bw {
namespace tree {

// Rows of a block, in tiles of eight.
static int tiles_of_eight(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

constexpr int kFewRows = 32;            // query rows of a head that the mma.sync kernel takes
constexpr int kMaxCluster = 8;
constexpr int kCut = 512;               // positions of a warp, where contexts are long: their lengths differ, and the last block is waited for
// Blocks that share a context of a (sequence, head, row tile), a multiple of eight where more than a cluster.
// The fewest waves of two blocks per SM times what a block takes: the tiles of 16 positions that a warp is left with (0.45 us for eight columns) and 0.9 us
// for a cluster's merge; clusters of other than 2, 4 or 8 blocks take longer to be placed, and in a wave that is nearly full not all find a place.  Four tiles of
// columns, bound by mma.sync: one wave (32 x 10 nodes, 1,500 positions: 83 us, in three shares 109).
// At least as many as leave a warp kCut positions, as far as the records allow (rows of few heads: any number, scratch_bytes; many rows: two waves of
// blocks).  Still more shares of a long context, joined by a second launch, where a wave has room for them.
// Measured (us, 32 / 8 heads, fp32; in 1 2 3 4 5 6 8 shares): 1 x 100 positions of 8 bits 3.9 5.1 5.3 5.7 5.9 6.0 6.1, 1 x 500 6.1 5.9 6.0 5.5 5.6 5.7 5.7, 1 x 2,048
// 13.7 10.0 8.8 7.7 7.6 7.3 6.7, 8 x 4,000 24 20 17 15 22 22 21, 20 x 6,000 48 47 41 44 43 48 54, 32 x 8,192 75 74 75 76 79 85 95; 4 trees of 8 nodes,
// 1,000 positions of 16 bits, 28 / 4 heads, 25.6 20.4 18.4 16.6 15.7 15.9 13.9.  Clusters of 16 need 16 free SMs next to each other: 1 x 2,048 positions
// with 64 rows 27 us, as two clusters of 8 and a merge 20.
static int choose_splits(long pairs, int ctx, int slots, int warps, int nt, bool few) {
    const long tiles = (ctx + kTile - 1) / kTile, least = (ctx + (long)kCut * warps - 1) / (kCut * warps);
    auto cost = [&](long k) {
        const bool whole = (k & (k - 1)) == 0;
        long waves = (pairs * k + slots - 1) / slots;
        if (!whole && nt == 1 && pairs * k * 20 > (20 * waves - 3) * slots) ++waves;
        return waves * ((tiles + k * warps - 1) / (k * warps) * nt + (k == 1 ? 0 : whole ? 2 : 3));
    };
    long n = least < 1 ? 1 : least > kMaxCluster ? kMaxCluster : least;
    for (long k = n + 1; k <= kMaxCluster && k * warps < tiles + warps && (nt < 4 || pairs * k <= slots); ++k)
        if (cost(k) < cost(n)) n = k;
    if (n == kMaxCluster) {
        const long room = slots / pairs, most = ctx / (32 * warps), more = (room < most ? room : most) / kMaxCluster * kMaxCluster;
        if (more > n) n = more;
        if (n < least) {
            n = (least + kMaxCluster - 1) / kMaxCluster * kMaxCluster;
            const long records = 2L * slots / pairs;
            if (!few && n > records) n = records < kMaxCluster ? kMaxCluster : records / kMaxCluster * kMaxCluster;
        }
    }
    return (int)n;
}

template <int NT, bool kCoded, typename A, bool kPair = false>
static cudaError_t launch(Args a, int ctx, void* scratch, size_t scratch_bytes, cudaStream_t st) {
    using Sh = Shape<NT, kCoded>;
    auto kern = attend_kernel<NT, kCoded, A, kPair>;
    static std::once_flag once[kMaxDevices];
    const int dev = current_device();
    std::call_once(once[dev], [&] {
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
        cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    a.nsplit = choose_splits((long)a.M * a.c.heads * a.tiles, ctx, 2 * sm_count(dev), Sh::kWarps, NT, a.rows <= kFewRows);
    a.cluster = a.nsplit <= kMaxCluster ? a.nsplit : kMaxCluster;
    const int groups = a.nsplit / a.cluster;
    if (groups > 1) {
        if (!scratch || scratch_bytes < (size_t)a.M * a.c.heads * a.rows * groups * kPart * sizeof(float)) return cudaErrorInvalidValue;
        a.part = static_cast<float*>(scratch);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.nsplit, a.c.heads * a.tiles, a.M);
    cfg.blockDim = dim3(Sh::kWarps * 32);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    count_launch(1);
    if (e == cudaSuccess && groups > 1) {
        const long rows = (long)a.M * a.c.heads * a.rows;
        e = launch_pdl(attend_merge_kernel<A>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
        count_launch(1);
    }
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
template <bool kCoded, typename A>
static cudaError_t launch_rows(const Args& a, int nt, int ctx, void* scratch, size_t bytes, cudaStream_t st) {
    if (sizeof(A) == 4 && a.rows <= 4) return launch<1, kCoded, float, true>(a, ctx, scratch, bytes, st);
    return nt == 1 ? launch<1, kCoded, A>(a, ctx, scratch, bytes, st) : nt == 2 ? launch<2, kCoded, A>(a, ctx, scratch, bytes, st)
                                                                                : launch<4, kCoded, A>(a, ctx, scratch, bytes, st);
}

template <bool kTall, bool kCoded, typename A>
static cudaError_t launch_tc(const Args& a, cudaStream_t st) {
    auto kern = attend_tc_kernel<kTall, kCoded, A>;
    constexpr int smem = TcShape<kTall, kCoded, sizeof(A) == 4>::kSmem;
    static std::once_flag once[kMaxDevices];
    std::call_once(once[current_device()], [&] { cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    cudaError_t e = launch_pdl(kern, dim3(a.blocks), dim3(kTcThreads), smem, st, a);
    count_launch(1);
    if (e == cudaSuccess && a.flat) {
        e = launch_pdl(attend_tc_merge_kernel<A>, dim3((a.rows + 31) / 32 * 2, a.c.heads, a.M), dim3(256), 0, st, a);
        count_launch(1);
    }
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
template <bool kCoded, typename A>
static cudaError_t launch_tc_rows(const Args& a, cudaStream_t st) {
    return a.group_rows > 128 ? launch_tc<true, kCoded, A>(a, st) : launch_tc<false, kCoded, A>(a, st);
}

// Which kernel.  The tcgen05 kernel takes some 20 us before it pays (queries into shared memory, the pipeline's start, records and their merge); a
// tile of the mma.sync kernel (32 rows, 16 positions) takes a block 0.4 us.  So: by the tiles that an SM gets.  One or two row tiles leave the 128
// lanes of an accumulator half empty, the more so the more heads there are to begin with.  Measured (us, mma.sync / tcgen05; 32 / 8 heads, fp32, 8 bits): 64
// nodes, 8 x 2,048 positions 152 / 60, 4 x 1,000 40 / 32, 4 x 300 20 / 28; 24 nodes, 8 x 2,048 55 / 39, 4 x 1,000 22 / 26; 16 nodes, 32 x 1,000 67 / 70,
// 8 x 5,310 83 / 63; 10 nodes, 8 x 1,300 29 / 30, 8 x 3,000 53 / 43, 32 x 400 35 / 46; 8 nodes, 32 x 4,000 119 / 148.  More than 64 rows: contexts of up to
// two tiles stay whole in a block, without records and merge (64 nodes, 8 x 60 positions 25 / 16, 16 x 60 46 / 16), longer ones are laid in a line (8 x 100
// 28 / 31, 8 x 200 31 / 32, 8 x 300 36 / 34, 16 x 128 51 / 39, 4 x 128 16 / 28, 4 x 600 29 / 30): the step from 16 to 80 tiles.
static bool many_rows(long heads, int rows, int ctx, int sms) {
    if (rows <= kFewRows) return false;
    const double tiles = (double)heads * ((rows + 31) / 32) * ((ctx + 15) / 16) / sms;
    return tiles >= (rows <= 64 ? 60 + 0.8 * heads : ctx <= 2 * kTcKeys ? 16 : 80);
}
static int g_route = 0;   // experiments: 1 mma.sync, 2 tcgen05
void set_route(int v) { g_route = v; }

}  // namespace tree
}  // namespace bw

using namespace bw;

namespace bw {
namespace tree {
// Scratch of the tcgen05 kernel: the line of work, two records per block, the sums that fp32 activations keep.
constexpr size_t kLineBytes = 4096;
static size_t record_bytes(long blocks, int rows) { return (size_t)2 * blocks * rows * kPart * sizeof(float); }
static size_t kept_bytes(long blocks) { return (size_t)blocks * 2 * kHd * 128 * sizeof(float); }
}  // namespace tree
}  // namespace bw

// A bound for any smaller call too.  The blocks are at most as many as SMs; mma.sync kernel: records of 32 rows of two waves, or of long
// contexts' shares of four warps for rows of few heads.  tcgen05 kernel: where its rows are many enough, or it is forced.
extern "C" size_t bw_attention_tree_scratch_bytes(int M, int T, int num_q_heads, int num_kv_heads, int max_context) {
    if (M < 1 || T < 1 || T > tree::kMaxNodes || num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads || max_context < 1) return 0;
    const int sms = sm_count(current_device()), rows = T * (num_q_heads / num_kv_heads), few = rows < tree::kFewRows ? rows : tree::kFewRows;
    const size_t tc = tree::kLineBytes + tree::record_bytes(sms, rows < 256 ? rows : 256) + tree::kept_bytes(sms);
    const size_t need = rows <= tree::kFewRows && tree::g_route != 2 ? tree::record_bytes(sms, 32) : tc;
    const long positions = 4L * tree::kCut * tree::kMaxCluster, groups = ((long)max_context + positions - 1) / positions;
    const size_t shares = (size_t)M * num_kv_heads * few * groups * tree::kPart * sizeof(float);
    return groups > 1 && shares > need ? shares : need;
}

extern "C" int bw_attention_tree(void* out, const void* q, const bw_kv_cache* cache, const int* d_first_row,
                                 const unsigned long long* d_mask_or_null, const int* d_count_or_null, int ctx_hint, int num_q_heads, int M, int T,
                                 int bf16, void* scratch, size_t scratch_bytes, void* stream) {
    tree::Args a{};
    if (!kv::view(cache, &a.c) || !out || !q || !d_first_row || num_q_heads < 1 || num_q_heads % a.c.heads || M < 1 || M > 65535 || T < 1 ||
        T > tree::kMaxNodes || ctx_hint < 0)
        return cudaErrorInvalidValue;
    if (!kv::aligned(out, 16) || !kv::aligned(q, 16) || !kv::aligned(d_mask_or_null, 8) || !kv::aligned(scratch, 16)) return cudaErrorInvalidValue;
    a.out = out; a.q = q; a.first = d_first_row; a.count = d_count_or_null; a.mask = d_mask_or_null;
    a.nq = num_q_heads; a.M = M; a.T = T; a.group = num_q_heads / a.c.heads;
    if ((long)a.group * T > (1 << 20)) return cudaErrorInvalidValue;
    a.rows = a.group * T;
    const int ctx = ctx_hint > 0 && ctx_hint < a.c.max_seq ? ctx_hint : a.c.max_seq, sms = sm_count(current_device());
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tree::g_route == 2 || (tree::g_route == 0 && tree::many_rows((long)M * a.c.heads, a.rows, ctx, sms))) {
        a.group_rows = a.rows > 128 ? 256 : 128;
        a.groups = (a.rows + a.group_rows - 1) / a.group_rows;
        a.rec_rows = a.rows < a.group_rows ? a.rows : a.group_rows;
        const long pairs = (long)M * a.c.heads * a.groups, tiles = (ctx + tree::kTcKeys - 1) / tree::kTcKeys;
        if (pairs > (1L << 30) || a.c.heads > 65535) return cudaErrorInvalidValue;
        // In a line, unless every head's context is short or heads are many times the blocks.
        a.pairs = (int)pairs;
        a.flat = M <= tree::kPlanned && pairs < 4L * sms && tiles > 2 && pairs * (a.c.max_seq / tree::kTcKeys + 1) < (1L << 30);
        const long work = a.flat ? pairs * tiles / 2 : pairs;    // (two tiles for a block or more)
        a.blocks = (int)(work < sms ? work : sms);
        const size_t records = a.flat ? tree::kLineBytes + tree::record_bytes(a.blocks, a.rec_rows) : 0;
        if ((a.flat || !bf16) && (!scratch || scratch_bytes < records + (bf16 ? 0 : tree::kept_bytes(a.blocks)))) return cudaErrorInvalidValue;
        a.cum = static_cast<int*>(scratch);
        a.part = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + tree::kLineBytes);
        a.kept = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + records);
        a.status = status_word_ptr();
        if (a.c.coded()) return bf16 ? tree::launch_tc_rows<true, __nv_bfloat16>(a, st) : tree::launch_tc_rows<true, float>(a, st);
        return bf16 ? tree::launch_tc_rows<false, __nv_bfloat16>(a, st) : tree::launch_tc_rows<false, float>(a, st);
    }
    const int nt = tree::tiles_of_eight(a.rows);
    a.tiles = (a.rows + 8 * nt - 1) / (8 * nt);
    if ((long)a.c.heads * a.tiles > 65535) return cudaErrorInvalidValue;
    if (a.c.coded())
        return bf16 ? tree::launch_rows<true, __nv_bfloat16>(a, nt, ctx, scratch, scratch_bytes, st) : tree::launch_rows<true, float>(a, nt, ctx, scratch, scratch_bytes, st);
    return bf16 ? tree::launch_rows<false, __nv_bfloat16>(a, nt, ctx, scratch, scratch_bytes, st) : tree::launch_rows<false, float>(a, nt, ctx, scratch, scratch_bytes, st);
}
