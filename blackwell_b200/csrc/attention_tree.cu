// Attention of single tokens and of drafted trees over a binary16 or 8-bit cache (attention_tree.cuh): splits and entry points.
#include "attention_tree_tc.cuh"

#include <mutex>

#include "host_util.h"

namespace bw {
namespace tree {

constexpr int kMaxSplits = 64;

// Rows of a block, in tiles of eight.
static int tiles_of_eight(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// One wave of two blocks per SM, no split shorter than 256 positions.
static int choose_splits(long blocks, int ctx, int sms) {
    long n = 2L * sms / blocks;
    if (n > ctx / 256) n = ctx / 256;
    if (n > kMaxSplits) n = kMaxSplits;
    return n < 1 ? 1 : (int)n;
}

template <int NT, bool kCoded, typename A>
static cudaError_t launch(const Args& a, cudaStream_t st) {
    auto kern = attend_kernel<NT, kCoded, A>;
    constexpr int smem = Shape<NT, kCoded>::kSmem;
    static std::once_flag once[kMaxDevices];
    std::call_once(once[current_device()], [&] { cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    cudaError_t e = launch_pdl(kern, dim3(a.nsplit, a.c.heads * a.tiles, a.M), dim3(kWarps * 32), smem, st, a);
    count_launch(1);
    if (e == cudaSuccess && a.nsplit > 1) {
        const long rows = (long)a.M * a.c.heads * a.rows;
        e = launch_pdl(attend_merge_kernel<A>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
        count_launch(1);
    }
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
template <bool kCoded, typename A>
static cudaError_t launch_rows(const Args& a, int nt, cudaStream_t st) {
    return nt == 1 ? launch<1, kCoded, A>(a, st) : nt == 2 ? launch<2, kCoded, A>(a, st) : launch<4, kCoded, A>(a, st);
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
        const long rows = (long)a.M * a.c.heads * a.rows;
        e = launch_pdl(attend_tc_merge_kernel<A>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
        count_launch(1);
    }
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
template <bool kCoded, typename A>
static cudaError_t launch_tc_rows(const Args& a, cudaStream_t st) {
    return a.group_rows > 128 ? launch_tc<true, kCoded, A>(a, st) : launch_tc<false, kCoded, A>(a, st);
}

static int g_route = 0;   // experiments: 1 mma.sync, 2 tcgen05
void set_route(int v) { g_route = v; }

}  // namespace tree
}  // namespace bw

using namespace bw;

// At most two records per SM of a block's rows, whatever the call's sizes, and the line of work.
extern "C" size_t bw_attention_tree_scratch_bytes(int M, int T, int num_q_heads, int num_kv_heads, int max_context) {
    if (M < 1 || T < 1 || T > tree::kMaxNodes || num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads || max_context < 1) return 0;
    const int rows = T * (num_q_heads / num_kv_heads), rec = rows < 32 ? 32 : rows < 256 ? rows : 256;
    return (size_t)2 * sm_count(current_device()) * rec * tree::kPart * sizeof(float) + 4096;
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
    if (tree::g_route == 2 || (tree::g_route == 0 && a.rows > 32)) {
        a.group_rows = a.rows > 128 ? 256 : 128;
        a.groups = (a.rows + a.group_rows - 1) / a.group_rows;
        a.rec_rows = a.rows < a.group_rows ? a.rows : a.group_rows;
        const long pairs = (long)M * a.c.heads * a.groups, tiles = (ctx + tree::kTcKeys - 1) / tree::kTcKeys;
        if (pairs > 0x7FFFFFFFL) return cudaErrorInvalidValue;
        a.status = status_word_ptr();
        a.flat = M <= tree::kPlanned && pairs < 4L * sms && tiles > 2 && pairs * (a.c.max_seq / tree::kTcKeys + 1) < 0x7FFFFFFFL;
        a.blocks = (int)(!a.flat ? pairs : pairs * tiles < sms ? pairs * tiles : sms);
        if (a.flat) {
            if (!scratch || scratch_bytes < 4096 + (size_t)2 * a.blocks * a.rec_rows * tree::kPart * sizeof(float)) return cudaErrorInvalidValue;
            a.cum = static_cast<int*>(scratch);
            a.part = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + 4096);
        }
        if (a.c.coded()) return bf16 ? tree::launch_tc_rows<true, __nv_bfloat16>(a, st) : tree::launch_tc_rows<true, float>(a, st);
        return bf16 ? tree::launch_tc_rows<false, __nv_bfloat16>(a, st) : tree::launch_tc_rows<false, float>(a, st);
    }
    const int nt = tree::tiles_of_eight(a.rows);
    a.tiles = (a.rows + 8 * nt - 1) / (8 * nt);
    if ((long)a.c.heads * a.tiles > 65535) return cudaErrorInvalidValue;
    a.nsplit = tree::choose_splits((long)M * a.c.heads * a.tiles, ctx, sms);
    if (a.nsplit > 1) {
        if (!scratch || scratch_bytes < (size_t)M * a.c.heads * a.rows * a.nsplit * tree::kPart * sizeof(float)) return cudaErrorInvalidValue;
        a.part = static_cast<float*>(scratch);
    }
    if (a.c.coded()) return bf16 ? tree::launch_rows<true, __nv_bfloat16>(a, nt, st) : tree::launch_rows<true, float>(a, nt, st);
    return bf16 ? tree::launch_rows<false, __nv_bfloat16>(a, nt, st) : tree::launch_rows<false, float>(a, nt, st);
}
