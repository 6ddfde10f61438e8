// Attention of the rows of a tree of drafted tokens over the paged cache.
//
//   out_t = sum_j softmax_j(scale q_t . k_j) v_j   over j < ctx and those j = ctx + i whose bit i the row's mask has
//
// One warp a row and head, each lane four of the 128 dimensions, the running maximum and sum of the softmax in registers.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tree_step.h"

namespace b200 {
namespace {

constexpr int kD = 128;

__global__ void __launch_bounds__(256)
tree_attn_kernel(const b200_tree_attn_args a, float scale_log2) {
  griddep_wait();
  const int s = blockIdx.z, head = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (head >= a.q_heads) return;
  const tree::Request r = tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_tree);
  const int* table = a.block_tables + static_cast<size_t>(s) * a.ld_tables;
  const int kv_head = head / (a.q_heads / a.kv_heads);
  const __nv_bfloat16* kv = static_cast<const __nv_bfloat16*>(a.kv_layer);
  for (int i = blockIdx.x; i < r.rows; i += gridDim.x) {
    const size_t row = r.row0 + i;
    const uint2 qw = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + row * a.ldq + head * kD + lane * 4);
    auto unpack = [](uint2 u, float* f) {
      f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xffff0000u), f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xffff0000u);
    };
    float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
    unpack(qw, q);
    for (int p = 0; p < r.ctx + r.rows; ++p) {
      const int j = p - r.ctx;
      if (j >= 0) {
        if (a.masks ? j >= 32 * a.words || !(static_cast<unsigned>(a.masks[row * a.words + (j >> 5)]) >> (j & 31) & 1) : j > i) continue;
      }
      const long long at = tree::cache_row(table, p, a.num_pages);
      float k[4] = {}, v[4] = {};
      if (at >= 0) {
        const __nv_bfloat16* base = kv + (((at >> 4) * 2 * a.kv_heads + kv_head) * 16 + (at & 15)) * kD + lane * 4;
        unpack(*reinterpret_cast<const uint2*>(base), k);
        unpack(*reinterpret_cast<const uint2*>(base + static_cast<size_t>(a.kv_heads) * 16 * kD), v);
      }
      float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      x *= scale_log2;
      const float top = fmaxf(m, x), shift = top == -INFINITY ? 0.f : top, old = exp2f(m - shift), w = exp2f(x - shift);
      m = top;
      l = l * old + w;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = o[d] * old + w * v[d];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 y;
    y.x = pack_bf16x2(o[0] * inv, o[1] * inv);
    y.y = pack_bf16x2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + row * a.ldo + head * kD + lane * 4) = y;
  }
}

}  // namespace

int paged_attention_tree(const b200_tree_attn_args& a, cudaStream_t st) {
  launch_pdl(tree_attn_kernel, dim3(std::min(a.max_tree, a.T), (a.q_heads + 7) / 8, a.S), dim3(256), 0, st, a, a.scale * 1.4426950408889634f);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
