// The cache that bw_kv_cache describes: rows of 128 in binary16, or in e4m3 codes with an fp32 scale per row.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/blackwell_b200.h"

namespace bw {
namespace kv {

constexpr int kHd = 128;
constexpr float kCodeMax = 448.f;       // largest e4m3 value
constexpr float kTinyRow = 1e-10f;      // rows with no larger element keep scale 1, as the int8 rule has it

// A cache seen from one layer: element offsets of sequence m and head g as in bw_kv_cache; scales at element / 128.
struct View {
    unsigned char *k, *v;
    float *ks, *vs;                     // NULL: binary16
    int heads, max_seq;
    size_t batch, layer;                // elements
    __host__ __device__ bool coded() const { return ks != nullptr; }
    // Sequences that are written must not share rows.
    __host__ bool apart(long sequences) const { return sequences == 1 || batch / kHd >= (size_t)heads * max_seq; }
    __host__ __device__ size_t row(int m, int g, long t) const { return (size_t)m * (batch / kHd) + layer / kHd + (size_t)g * max_seq + t; }
};

// Whether the description can be used; `out` is its view.
inline bool view(const bw_kv_cache* c, View* out) {
    if (!c || !c->k || !c->v || c->kv_heads < 1 || c->max_seq < 1) return false;
    if ((c->k_scale == nullptr) != (c->v_scale == nullptr)) return false;
    if (c->batch_elems % kHd || c->layer_elems % kHd) return false;
    if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) != 0) return false;
    if (((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) != 0) return false;
    *out = View{static_cast<unsigned char*>(c->k), static_cast<unsigned char*>(c->v), c->k_scale, c->v_scale, c->kv_heads, c->max_seq,
                c->batch_elems, c->layer_elems};
    return true;
}
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace kv
}  // namespace bw
