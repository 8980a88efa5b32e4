// Attention of single tokens and of drafted trees over a binary16 or 8-bit cache (attention_tree.cuh): splits and entry points.
#include "attention_tree.cuh"

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

}  // namespace tree
}  // namespace bw

using namespace bw;

// At most two blocks per SM of up to 32 rows write records, whatever the call's sizes.
extern "C" size_t bw_attention_tree_scratch_bytes(int M, int T, int num_q_heads, int num_kv_heads, int max_context) {
    if (M < 1 || T < 1 || T > tree::kMaxNodes || num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads || max_context < 1) return 0;
    return (size_t)2 * sm_count(current_device()) * 32 * tree::kPart * sizeof(float);
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
    const int nt = tree::tiles_of_eight(a.rows);
    a.tiles = (a.rows + 8 * nt - 1) / (8 * nt);
    if ((long)a.c.heads * a.tiles > 65535) return cudaErrorInvalidValue;
    const int ctx = ctx_hint > 0 && ctx_hint < a.c.max_seq ? ctx_hint : a.c.max_seq;
    a.nsplit = tree::choose_splits((long)M * a.c.heads * a.tiles, ctx, sm_count(current_device()));
    if (a.nsplit > 1) {
        if (!scratch || scratch_bytes < (size_t)M * a.c.heads * a.rows * a.nsplit * tree::kPart * sizeof(float)) return cudaErrorInvalidValue;
        a.part = static_cast<float*>(scratch);
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.c.coded()) return bf16 ? tree::launch_rows<true, __nv_bfloat16>(a, nt, st) : tree::launch_rows<true, float>(a, nt, st);
    return bf16 ? tree::launch_rows<false, __nv_bfloat16>(a, nt, st) : tree::launch_rows<false, float>(a, nt, st);
}
