// Norms of queries and keys for each head, rotary positions, and keys and values into the paged cache, in one pass.
//
//   y = x w / sqrt(mean(x^2) + eps);   (y_a, y_b) -> gain (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * freq
//
// Everything between the loads and the stores is fp32 and rounded once to bf16 (the norm's result is not rounded ahead of the rotation).  An angle of a far position
// has many turns: the frequency becomes a 64-bit part of a turn, and the product with the position drops whole turns by itself.  An angle of N turns is then off by N 2^-52 (the frequency in
// turns, in fp64: 2^-35 of a turn at position 10^6, 2^-23.6 at 2^31) and, as what is left of a turn goes to the sine in fp32, 2^-26 of a turn; an fp32 product would be off by 0.06 radians at position 10^6.
// A CTA has a token; its first threads make the token's cosines and sines while the heads are on their way.  Sixteen lanes have a head, eight values each in two
// pieces of four that hold both values of their pairs: (j, j + n / 4) where halves pair up, (2 j, 2 j + 1) where neighbours do.  Halves of a number of pairs that four does not
// divide go through shared memory.
// Memory bounds it: 8191 rows of 32 + 8 + 8 heads are 201 MB in and out, 41.1 us, 4.9 TB/s of 6.55 that a copy reaches (42.8 when values went
// through the norm's sums as well; two values an instruction took 63 registers, not 45, and 46 us).  Four rows are a launch and three dependent trips (slot and position, heads,
// stores), 3.1 us; 999 rows 4.6.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "beam_step.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kAhead = 3, kD = 128;      // kAhead: heads of a thread on their way
constexpr int kManyRows = 2048;          // rows from which on a CTA has 128 threads for its row, not 256: 8191 rows 47.2 us -> 42.8, four rows 3.1 -> 4.1

struct Piece {
  float v[4];
};
__device__ __forceinline__ Piece widen(uint2 u) {
  return {__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
}

// kStaged: halves of a number of pairs that four does not divide
template <bool kStaged, int kThreads>
__global__ void __launch_bounds__(kThreads)
norm_rope_kernel(const b200_norm_rope_args a) {
  constexpr int kWarps = kThreads / 32;
  __shared__ float2 turn[kD / 2];
  __shared__ float stage[kStaged ? kWarps * 2 : 1][kD];
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = lane & 15, n = a.dims / 2;
  griddep_enter();
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.qkv) + static_cast<size_t>(t) * a.ldx;
  const int slot = a.slots[t], heads = a.q_heads + 2 * a.kv_heads, turned = a.q_heads + a.kv_heads;
  const bool kept = slot >= 0 && (slot >> 4) < a.num_pages;
  // this lane's pieces of a head
  const bool beside = a.interleaved || kStaged;
  const int p0 = beside ? 2 * j : j < n / 4 ? j : 2 * j, p1 = beside ? 2 * j + 1 : j < n / 4 ? j + n / 4 : 2 * j + 1;
  bool first = true;
  int h0 = warp * 2 + (lane >> 4);
  do {      // once for every warp: one that has no heads has pairs of the table
    uint2 u0[kAhead], u1[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int h = h0 + 2 * kWarps * k;
      u0[k] = u1[k] = make_uint2(0, 0);
      if (h < heads) {
        u0[k] = reinterpret_cast<const uint2*>(x + h * kD)[p0];
        u1[k] = reinterpret_cast<const uint2*>(x + h * kD)[p1];
      }
    }
    if (first) {
      if (tid < n) {
        const double turns = a.freqs[tid] * 0.15915494309189533577;      // of a position
        const long long part = static_cast<long long>(static_cast<unsigned long long>(__double2ll_rn((turns - rint(turns)) * 18446744073709551616.0)) * static_cast<unsigned long long>(static_cast<long long>(a.positions[t])));
        float s, c;
        sincospif(__ll2float_rn(part) * 1.0842021724855044e-19f, &s, &c);      // 2^-63: in half turns
        turn[tid] = make_float2(c * a.gain, s * a.gain);
      }
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int h = h0 + 2 * kWarps * k;
      if (h - (lane >> 4) >= heads) break;      // for both halves of the warp
      uint2 r0 = u0[k], r1 = u1[k];      // values pass as they are, odd ones too
      if (h - (lane >> 4) < turned) {
        Piece y0 = widen(u0[k]), y1 = widen(u1[k]);
        const void* w = h < a.q_heads ? a.q_norm : a.k_norm;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += y0.v[i] * y0.v[i] + y1.v[i] * y1.v[i];
#pragma unroll
        for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (h < turned && w) {
          const float inv = rsqrtf(sum * (1.f / kD) + a.eps);
          const size_t at = static_cast<size_t>(h < a.q_heads ? h * a.q_norm_ld : (h - a.q_heads) * a.k_norm_ld);
          Piece w0, w1;
          if (a.norm_f32) {
            const float4 f0 = reinterpret_cast<const float4*>(static_cast<const float*>(w) + at)[p0], f1 = reinterpret_cast<const float4*>(static_cast<const float*>(w) + at)[p1];
            w0 = {f0.x, f0.y, f0.z, f0.w};
            w1 = {f1.x, f1.y, f1.z, f1.w};
          } else {
            w0 = widen(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at)[p0]);
            w1 = widen(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at)[p1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y0.v[i] *= inv * w0.v[i];
            y1.v[i] *= inv * w1.v[i];
          }
        }
        if (kStaged) {
          float* row = stage[warp * 2 + (lane >> 4)];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            row[4 * p0 + i] = y0.v[i];
            row[4 * p1 + i] = y1.v[i];
          }
          __syncwarp();
          if (h < turned) {
            auto turn_one = [&](int d, float& y) {
              if (d >= 2 * n) return;
              const float2 cs = turn[d < n ? d : d - n];
              y = d < n ? y * cs.x - row[d + n] * cs.y : y * cs.x + row[d - n] * cs.y;
            };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              turn_one(4 * p0 + i, y0.v[i]);
              turn_one(4 * p1 + i, y1.v[i]);
            }
          }
        } else if (h < turned) {
          if (a.interleaved) {
            auto turn_pair = [&](int pair, float& y, float& z) {
              if (pair >= n) return;
              const float2 cs = turn[pair];
              const float was = y;
              y = was * cs.x - z * cs.y;
              z = z * cs.x + was * cs.y;
            };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              turn_pair(2 * p0 + i, y0.v[2 * i], y0.v[2 * i + 1]);
              turn_pair(2 * p1 + i, y1.v[2 * i], y1.v[2 * i + 1]);
            }
          } else if (j < n / 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 cs = turn[4 * j + i];
              const float was = y0.v[i];
              y0.v[i] = was * cs.x - y1.v[i] * cs.y;
              y1.v[i] = y1.v[i] * cs.x + was * cs.y;
            }
          }
        }
        if (h < turned) {
          r0 = make_uint2(pack_bf16x2(y0.v[0], y0.v[1]), pack_bf16x2(y0.v[2], y0.v[3]));
          r1 = make_uint2(pack_bf16x2(y1.v[0], y1.v[1]), pack_bf16x2(y1.v[2], y1.v[3]));
        }
      }
      uint2* to = nullptr;
      if (h < a.q_heads) to = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(t) * a.ldo + h * kD);
      else if (h < heads && kept)      // a page has the heads' keys one behind the other, then the values
        to = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.kv_layer) + ((static_cast<size_t>(slot >> 4) * 2 * a.kv_heads + (h - a.q_heads)) * 16 + (slot & 15)) * kD);
      if (to) {
        to[p0] = r0;
        to[p1] = r1;
      }
    }
    h0 += 2 * kWarps * kAhead;
  } while (h0 - (lane >> 4) < heads);
}

}  // namespace

int norm_rope_kv_write(const b200_norm_rope_args& a, cudaStream_t st) {
  const bool staged = !a.interleaved && a.dims % 8 != 0;
  if (a.T >= kManyRows) launch_pdl(staged ? norm_rope_kernel<true, 128> : norm_rope_kernel<false, 128>, dim3(a.T), dim3(128), 0, st, a);
  else launch_pdl(staged ? norm_rope_kernel<true, 256> : norm_rope_kernel<false, 256>, dim3(a.T), dim3(256), 0, st, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
