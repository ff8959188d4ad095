// Single-token attention over the paged 8-bit KV cache (layout in paged_sm100.cuh).
//
// Per request b with n cached tokens (the query's own among them) and query head h of KV head g:
//   q' = R(n - 1) q            s_j = (q' . k8_j) ks[page_j, g] scale       j < n
//   out = sum_j softmax(s)_j v8_j vs[page_j, g]
// The cached keys are rotated already. A request without tokens gives zeros.
#pragma once

#include "paged_sm100.cuh"

namespace du {

struct DecodePagedParams {
  const void* q;        // [B, Hq, D]
  const uint8_t* k8;    // [N, Hkv, block, D] e4m3
  const uint8_t* v8;
  const float* ks;      // [N, Hkv]
  const float* vs;
  const int* table;     // [B, width]
  const int* lens;      // [B]
  const void* cos;      // [positions, D/2]
  const void* sin;
  void* out;            // [B, Hq, D]
  long long positions;
  int B, Hq, Hkv, N, block, width;
  float scale_log2;
};

// One CTA per (query head, request); a warp takes a key at a time, a lane the row's elements
// lane, lane + 32, ...; running maximum and sum per warp, joined at the end.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) decode_paged_kernel(const DecodePagedParams p) {
  constexpr int EPL = (D + 31) / 32;
  constexpr int NW = 8;
  __shared__ float sm_q[D], sm_o[NW][D], sm_m[NW], sm_l[NW];
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / (p.Hq / p.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = p.lens[b];
  if (n < 0 || n > p.width * p.block || n > p.positions) {
    if (threadIdx.x == 0) record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(n));
    n = 0;
  }
  auto at16 = [&](const void* base, long long i) {
    if constexpr (BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
    else return __half2float(static_cast<const __half*>(base)[i]);
  };
  if (n > 0)
    for (int d = threadIdx.x; d < D / 2; d += 256) {
      const long long qr = (static_cast<long long>(b) * p.Hq + h) * D, tr = static_cast<long long>(n - 1) * (D / 2);
      const float x1 = at16(p.q, qr + d), x2 = at16(p.q, qr + D / 2 + d);
      const float c = at16(p.cos, tr + d), s = at16(p.sin, tr + d);
      sm_q[d] = (x1 * c - x2 * s) * p.scale_log2;
      sm_q[d + D / 2] = (x2 * c + x1 * s) * p.scale_log2;
    }
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
  for (int j = warp; j < n; j += NW) {
    const int id = p.table[static_cast<long long>(b) * p.width + j / p.block];
    if (id < 0 || id >= p.N) {
      if (lane == 0) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(id));
      m = __int_as_float(0x7fc00000);
      break;
    }
    const long long cell = static_cast<long long>(id) * p.Hkv + kvh;
    const long long row = (cell * p.block + j % p.block) * D;
    float dot = 0.f, vv[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int d = lane + 32 * e;
      vv[e] = 0.f;
      if (d < D) {
        dot = fmaf(sm_q[d], e4m3x2_widen(p.k8[row + d]).x, dot);
        vv[e] = e4m3x2_widen(p.v8[row + d]).x;
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = dot * p.ks[cell], mn = s > m ? s : m;
    const float a = ex2(m - mn), w = ex2(s - mn), wv = w * p.vs[cell];
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = acc[e] * a + wv * vv[e];
    m = mn;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e)
    if (lane + 32 * e < D) sm_o[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float M = -INFINITY, L = 0.f, A = 0.f;
    for (int w = 0; w < NW; ++w) M = (sm_m[w] > M || sm_m[w] != sm_m[w]) ? sm_m[w] : M;
    for (int w = 0; w < NW; ++w) {
      const float f = (sm_m[w] == -INFINITY && M == M) ? 0.f : ex2(sm_m[w] - M);
      L += sm_l[w] * f;
      A += sm_o[w][d] * f;
    }
    const float val = n > 0 ? A / L : 0.f;
    const long long o = (static_cast<long long>(b) * p.Hq + h) * D + d;
    if constexpr (BF16) static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(val);
    else static_cast<__half*>(p.out)[o] = __float2half_rn(val);
  }
}

}  // namespace du
