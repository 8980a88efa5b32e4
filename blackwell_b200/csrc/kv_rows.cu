// Rows of a KV cache: written from the QKV projection (head norm, rotation, quantising), moved between the beams of a search, and
// moved together once a path of a drafted tree has been accepted.
#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"
#include "host_util.h"
#include "kv_cache.cuh"
#include "lm_device.cuh"

namespace bw {
namespace kv {

// ------------------------------------------------------------------------------------------------------------------ writing
struct WriteArgs {
    void* q_out;
    View c;
    const void* qkv;
    const float *q_w, *k_w;
    const int *first, *offset, *count;
    int nq, M, T;
    float eps;
};
// base^(-2i/128) / 2 pi, i = 0..63: turns per position, as fractions of 2^64, right to 2^-55 (53-bit products on the host).  A position times one of them,
// modulo 2^64, is the angle to position * 2^-55 turns: in 32-bit floating point it would be off by position * 2^-24, visible from some thousand positions on.
struct Turns {
    unsigned long long f[kHd / 2];
};
// cos, sin of the angle.
__device__ __forceinline__ float2 turn_of(long long position, unsigned long long per) {
    const unsigned long long a = (unsigned long long)position * per;
    float s, c;
    sincospif((float)(int)(uint32_t)(a >> 32) * 0x1p-31f, &s, &c);
    return make_float2(c, s);
}

// A lane that warp_sum_many<N> leaves the sum of value j.
template <int N>
__device__ __forceinline__ constexpr int lane_of(int j) {
    int lane = 0;
    for (int w = N, off = 16; w > 1; w >>= 1, off >>= 1)
        if (j & (w / 2)) lane |= off;
    return lane;
}
// A warp takes HW heads of one row (token or node), four dimensions of each per lane.  x / sqrt(mean x^2 + eps) * w, then pairs
// (2i, 2i + 1) turned; a cached row is stored in binary16, or divided by absmax / 448 and rounded to e4m3.
constexpr int kWriteWarps = 12;         // warps of a block, at most
template <typename A, int HW>
__global__ void __launch_bounds__(kWriteWarps * 32, 3) write_rows_kernel(const WriteArgs a, const __grid_constant__ Turns turns) {
    __shared__ __align__(16) float2 s_turn[kHd / 2];                 // of the block's row, a pair of dimensions each
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, heads = a.nq + 2 * a.c.heads;
    const int m = blockIdx.x / (uint32_t)a.T, i = blockIdx.x - m * a.T, h0 = (blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5)) * HW;
    const size_t at = blockIdx.x;                       // row of the call
    const int first = a.first[m];
    if (first < 0 || (a.count && i >= a.count[m])) return;
    const A* x = static_cast<const A*>(a.qkv) + (at * heads + h0) * kHd + 4 * lane;
    float4 v[HW];
#pragma unroll
    for (int j = 0; j < HW; ++j) v[j] = h0 + j < heads ? lm::load4(x + j * kHd) : make_float4(0.f, 0.f, 0.f, 0.f);
    const int turned = a.nq + a.c.heads;                // heads that are normed and turned
    for (int e = threadIdx.x; e < kHd / 2; e += blockDim.x)
        s_turn[e] = turn_of((long long)first + (a.offset ? a.offset[at] : i), turns.f[e]);
    __syncthreads();
    if (h0 < turned) {
        float4 qw = make_float4(1.f, 1.f, 1.f, 1.f), kw = qw;
        if (a.q_w && h0 < a.nq) qw = *reinterpret_cast<const float4*>(a.q_w + 4 * lane);
        if (a.k_w && h0 + HW > a.nq) kw = *reinterpret_cast<const float4*>(a.k_w + 4 * lane);
        const float4 turn = *reinterpret_cast<const float4*>(&s_turn[2 * lane]);
        const float2 r0 = make_float2(turn.x, turn.y), r1 = make_float2(turn.z, turn.w);
        float ss[HW];
#pragma unroll
        for (int j = 0; j < HW; ++j) ss[j] = fmaf(v[j].w, v[j].w, fmaf(v[j].z, v[j].z, fmaf(v[j].y, v[j].y, v[j].x * v[j].x)));
        // a lane ends up with the sum of one of the heads, and gives its root to all
        const float root = rsqrtf(warp_sum_many<HW>(ss, lane) / 128.0f + a.eps);
#pragma unroll
        for (int j = 0; j < HW; ++j) {
            const int h = h0 + j;
            if (h >= turned) break;
            const bool is_q = h < a.nq;
            float4 y = v[j];
            if (is_q ? a.q_w != nullptr : a.k_w != nullptr) {
                const float is = __shfl_sync(0xffffffffu, root, lane_of<HW>(j));
                const float4 g = is_q ? qw : kw;
                y = make_float4(y.x * is * g.x, y.y * is * g.y, y.z * is * g.z, y.w * is * g.w);
            }
            v[j] = make_float4(fmaf(y.x, r0.x, -(y.y * r0.y)), fmaf(y.x, r0.y, y.y * r0.x), fmaf(y.z, r1.x, -(y.w * r1.y)),
                               fmaf(y.z, r1.y, y.w * r1.x));
        }
    }
    const long row = (long)first + i;
#pragma unroll
    for (int j = 0; j < HW; ++j) {
        const int h = h0 + j;
        if (h >= heads) break;
        const float4 y = v[j];
        if (h < a.nq) {
            lm::store4(static_cast<A*>(a.q_out) + (at * a.nq + h) * kHd + 4 * lane, y);
            continue;
        }
        if (row >= a.c.max_seq) continue;               // a row outside of the cache is never written
        const bool is_k = h < turned;
        const size_t to = a.c.row(m, h - a.nq - (is_k ? 0 : a.c.heads), row);
        unsigned char* side = is_k ? a.c.k : a.c.v;
        if (!a.c.coded()) {
            const __half2 lo = __floats2half2_rn(y.x, y.y), hi = __floats2half2_rn(y.z, y.w);
            *reinterpret_cast<uint2*>(side + (to * kHd + 4 * lane) * 2) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
            const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))))));
            const bool tiny = top < kTinyRow;
            // 448 / top to 2^-22: which of two codes is nearer changes for one element in a million (divided exactly, 8 x 512 rows take 2 % longer).  A
            // quarter of both: the fast division gives zero for divisors above 2^126.
            const float up = tiny ? 1.f : __fdividef(0.25f * kCodeMax, 0.25f * top);
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y.x * up, y.y * up), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y.z * up, y.w * up), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint32_t*>(side + to * kHd + 4 * lane) = lo | hi << 16;
            if (lane == 0) (is_k ? a.c.ks : a.c.vs)[to] = tiny ? 1.f : top * (1.0f / kCodeMax);
        }
    }
}

template <typename A>
static cudaError_t write_launch(const WriteArgs& a, const Turns& turns, cudaStream_t st) {
    const int heads = a.nq + 2 * a.c.heads;
    const long rows = (long)a.M * a.T;
    // A block has a row, or part of its heads.  Few rows: a head per warp and two warps per block, everything is latency.  Many: four heads per
    // warp.  Measured (8 x 512 rows, 32 / 8 heads, fp32 to 8 bits, 176 MB): 32.2 us, 5.5 TB/s; with the angles formed by every warp 34.3, in 64-bit
    // floating point 37.6; eight heads per warp leave too few warps (44).
    const bool many = rows * heads > 32L * sm_count(current_device());
    const int per_row = many ? (heads + 3) / 4 : heads, warps = many ? (per_row < kWriteWarps ? per_row : kWriteWarps) : 2;
    const long parts = (per_row + warps - 1) / warps;
    if (rows > 0x7FFFFFFFL || parts > 65535) return cudaErrorInvalidValue;
    const cudaError_t e = launch_pdl(many ? write_rows_kernel<A, 4> : write_rows_kernel<A, 1>, dim3((unsigned)rows, (unsigned)parts), dim3(warps * 32), 0, st, a, turns);
    count_launch(1);
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}

// ------------------------------------------------------------------------------------------------------------------ moving
struct MoveArgs {
    View c;
    size_t layer_stride;                // rows
    int layers;
    const int *index, *from, *to;       // parents / path; rows [from, to) / first row and count
    int n;                              // beams / most rows of a path
};
constexpr int kMaxBeams = 32, kMaxPath = 64;

// Sequence m * beams + b takes the rows [from, to) of m * beams + parent[b].  A thread owns 16 bytes of a row (and the row's scale,
// the first of them) in all beams of a group: it reads what every changed beam gets, then writes, so that parents may change too.  Bound by
// memory: 32 beams of 1,500 binary16 rows, 6 layers, 8 heads, 1.5 GB read and written: 232 us, 6.4 TB/s.
template <int NB>
__global__ void __launch_bounds__(256) reorder_kernel(const MoveArgs a) {
    pdl_trigger();
    pdl_wait();
    const int m = blockIdx.z, side = blockIdx.y & 1, plane = blockIdx.y >> 1;
    const int layer = plane / a.c.heads, g = plane - layer * a.c.heads;
    const int lo = a.from ? max(a.from[m], 0) : 0, hi = min(a.to[m], a.c.max_seq);
    const bool coded = a.c.coded();
    const int cols = coded ? 8 : 16;                    // 16-byte pieces of a row
    uint4* data = reinterpret_cast<uint4*>(side ? a.c.v : a.c.k);
    float* scale = side ? a.c.vs : a.c.ks;
    int parent[NB];
    bool any = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int p = b < a.n ? a.index[m * a.n + b] : b;
        parent[b] = p >= 0 && p < a.n && p != b ? p : -1;
        any |= parent[b] >= 0;
    }
    if (!any) return;
    const size_t base = a.c.row(m * a.n, g, 0) + layer * a.layer_stride, seq = a.c.batch / kHd;
    for (long u = (long)blockIdx.x * 256 + threadIdx.x; u < ((long)hi - lo) * cols; u += (long)gridDim.x * 256) {
        const long r = u / cols;
        const int col = (int)(u - r * cols);
        const size_t row = base + lo + r;
        uint4 x[NB];
        float s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (parent[b] >= 0) {
                x[b] = data[(row + parent[b] * seq) * cols + col];
                if (coded && col == 0) s[b] = scale[row + parent[b] * seq];
            }
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (parent[b] >= 0) {
                data[(row + b * seq) * cols + col] = x[b];
                if (coded && col == 0) scale[row + b * seq] = s[b];
            }
    }
}

// Row first + i takes row first + path[i], i < count: a warp has a plane (one side of a head in a layer).  Each step reads 128 pieces of 16
// bytes before it writes them.  An ascending path (path[i] >= i, each larger than the one before: the nodes of a tree in order) can go on so, because
// a later step reads behind all that is written; any other one is read whole first, through local memory.  32 paths of 2 to 11 rows in 576 planes
// of 8 bits, 37 MB: 11.8 us, 3.1 TB/s, mostly the latency of path, read and write (a block per plane that held a whole path in registers: 28).
__device__ __forceinline__ void keep_plane(const MoveArgs& a, uint4* data, float* scale, size_t base, const int* path, int first, int n, int lane) {
    const int shift = scale ? 3 : 4, cols = 1 << shift;  // pieces of a row: 8 or 16
    auto source = [&](int i) {                           // path[i], or -1 where row i stays as it is
        if (i >= n) return -1;
        const int p = path[i];
        return p >= 0 && p < a.n && p != i && (long)first + max(p, i) < a.c.max_seq ? p : -1;
    };
    bool ascending = true;
    if (n * cols > 128) {
        const int lo = lane < n ? path[lane] : 1 << 20, hi = lane + 32 < n ? path[lane + 32] : 1 << 20;
        const int lo_next = __shfl_down_sync(0xffffffffu, lo, 1), hi_next = __shfl_down_sync(0xffffffffu, hi, 1), hi_first = __shfl_sync(0xffffffffu, hi, 0);
        const bool fine = (lane >= n || (lo >= lane && lo < (lane < 31 ? lo_next : hi_first))) &&
                          (lane + 32 >= n || (hi >= lane + 32 && (lane == 31 || hi < hi_next)));
        ascending = __all_sync(0xffffffffu, fine);
    }
    if (ascending) {
        for (int u0 = 0; u0 < n * cols; u0 += 128) {
            uint4 x[4];
            float s[4];
            int p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = source((u0 + lane + 32 * j) >> shift);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = (lane + 32 * j) & (cols - 1);
                if (p[j] >= 0) {
                    x[j] = data[((base + p[j]) << shift) + col];
                    if (scale && col == 0) s[j] = scale[base + p[j]];
                }
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int u = u0 + lane + 32 * j, i = u >> shift, col = u & (cols - 1);
                if (p[j] >= 0) {
                    data[((base + i) << shift) + col] = x[j];
                    if (scale && col == 0) scale[base + i] = s[j];
                }
            }
            __syncwarp();
        }
        return;
    }
    uint4 x[kMaxPath * 16 / 32];
    float s[kMaxPath * 16 / 32];
#pragma unroll 1
    for (int j = 0; 32 * j < n * cols; ++j) {
        const int u = lane + 32 * j, p = source(u >> shift), col = u & (cols - 1);
        if (p >= 0) {
            x[j] = data[((base + p) << shift) + col];
            if (scale && col == 0) s[j] = scale[base + p];
        }
    }
    __syncwarp();
#pragma unroll 1
    for (int j = 0; 32 * j < n * cols; ++j) {
        const int u = lane + 32 * j, i = u >> shift, col = u & (cols - 1);
        if (source(i) >= 0) {
            data[((base + i) << shift) + col] = x[j];
            if (scale && col == 0) scale[base + i] = s[j];
        }
    }
}
__global__ void __launch_bounds__(256) keep_rows_kernel(const MoveArgs a) {
    pdl_trigger();
    pdl_wait();
    const int m = blockIdx.y, unit = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (unit >= 2 * a.layers * a.c.heads) return;
    const int first = a.from[m], n = min(a.to[m], a.n);
    if (first < 0 || n <= 0) return;
    const int side = unit & 1, plane = unit >> 1, layer = plane / a.c.heads, g = plane - layer * a.c.heads;
    uint4* data = reinterpret_cast<uint4*>(side ? a.c.v : a.c.k);
    float* scale = side ? a.c.vs : a.c.ks;
    const size_t base = a.c.row(m, g, first) + layer * a.layer_stride;
    const int* path = a.index + (size_t)m * a.n;
    keep_plane(a, data, scale, base, path, first, n, lane);
}

}  // namespace kv
}  // namespace bw

using namespace bw;

extern "C" int bw_qk_norm_rope_kv_rows(void* q_out, const bw_kv_cache* cache, const void* qkv, const float* q_norm_w_or_null,
                                       const float* k_norm_w_or_null, const int* d_first_row, const int* d_offset_or_null,
                                       const int* d_count_or_null, int num_q_heads, int M, int T, float eps, float rope_base, int bf16,
                                       void* stream) {
    kv::WriteArgs a{};
    if (!kv::view(cache, &a.c) || !a.c.apart(M) || !q_out || !qkv || !d_first_row || num_q_heads < 1 || M < 1 || T < 1 || !(rope_base > 0.f) || !(eps >= 0.f))
        return cudaErrorInvalidValue;
    if (!kv::aligned(q_out, 16) || !kv::aligned(qkv, 16) || !kv::aligned(q_norm_w_or_null, 16) || !kv::aligned(k_norm_w_or_null, 16))
        return cudaErrorInvalidValue;
    a.q_out = q_out; a.qkv = qkv; a.q_w = q_norm_w_or_null; a.k_w = k_norm_w_or_null;
    a.first = d_first_row; a.offset = d_offset_or_null; a.count = d_count_or_null;
    a.nq = num_q_heads; a.M = M; a.T = T; a.eps = eps;
    kv::Turns turns;
    const double ratio = pow((double)rope_base, -2.0 / kv::kHd);
    double f = 0.15915494309189535;                    // 1 / 2 pi
    for (int i = 0; i < kv::kHd / 2; ++i, f *= ratio) turns.f[i] = (unsigned long long)(long long)((f - floor(f)) * 0x1p63) << 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return bf16 ? kv::write_launch<__nv_bfloat16>(a, turns, st) : kv::write_launch<float>(a, turns, st);
}

// What both moves check of their planes: layers of layer_stride elements from the cache's own layer on.
static bool move_args(const bw_kv_cache* cache, long sequences, int layers, size_t layer_stride_elems, kv::MoveArgs* a) {
    if (!kv::view(cache, &a->c) || !a->c.apart(sequences) || layers < 1 || layer_stride_elems % kv::kHd) return false;
    const size_t plane = (size_t)a->c.heads * a->c.max_seq, stride = layer_stride_elems / kv::kHd, batch = a->c.batch / kv::kHd;
    if (layers > 1 && stride < plane) return false;
    // sequences around layers or layers around sequences, so that no two planes share rows
    if (layers > 1 && sequences > 1 && batch < (layers - 1) * stride + plane && stride < (sequences - 1) * batch + plane) return false;
    if (layers > (1 << 30) / (2 * (long)a->c.heads)) return false;
    a->layers = layers;
    a->layer_stride = layer_stride_elems / kv::kHd;
    return true;
}

extern "C" int bw_kv_reorder(const bw_kv_cache* cache, const int* d_parent, const int* d_from_or_null, const int* d_to, int beams, int M,
                             int layers, size_t layer_stride_elems, void* stream) {
    kv::MoveArgs a{};
    if (beams < 1 || beams > kv::kMaxBeams || M < 1 || M > 65535 || !move_args(cache, (long)M * beams, layers, layer_stride_elems, &a) || !d_parent || !d_to)
        return cudaErrorInvalidValue;
    a.index = d_parent; a.from = d_from_or_null; a.to = d_to; a.n = beams;
    const long planes = 2L * layers * a.c.heads;
    if (planes > 65535) return cudaErrorInvalidValue;
    const long most = ((long)a.c.max_seq * (a.c.coded() ? 8 : 16) + 255) / 256, fill = (32L * sm_count(current_device()) + planes * M - 1) / (planes * M);
    const dim3 grid((unsigned)(most < fill ? most : fill), (unsigned)planes, (unsigned)M);
    auto kern = beams <= 4 ? kv::reorder_kernel<4> : beams <= 8 ? kv::reorder_kernel<8> : beams <= 16 ? kv::reorder_kernel<16> : kv::reorder_kernel<32>;
    const cudaError_t e = launch_pdl(kern, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), a);
    count_launch(1);
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}

extern "C" int bw_kv_keep_rows(const bw_kv_cache* cache, const int* d_first_row, const int* d_path, const int* d_count, int M, int T, int layers,
                               size_t layer_stride_elems, void* stream) {
    kv::MoveArgs a{};
    if (!move_args(cache, M, layers, layer_stride_elems, &a) || !d_first_row || !d_path || !d_count || M < 1 || M > 65535 || T < 1 || T > kv::kMaxPath)
        return cudaErrorInvalidValue;
    a.index = d_path; a.from = d_first_row; a.to = d_count; a.n = T;
    const long planes = 2L * layers * a.c.heads;
    const cudaError_t e = launch_pdl(kv::keep_rows_kernel, dim3((unsigned)((planes + 7) / 8), (unsigned)M), dim3(256), 0, static_cast<cudaStream_t>(stream), a);
    count_launch(1);
    return e != cudaSuccess ? e : cudaPeekAtLastError();
}
