// Attention of several new tokens per request over the paged 8-bit KV cache (layout in
// paged_sm100.cuh).
//
// Request b has past_b tokens cached before its n_b = len_b - past_b new ones, which are cached too. For
// its new token t and query head h of KV head g:
//   q' = R(past_b + t) q    s_j = (q' . k8_j) ks[page_j, g] scale    j <= past_b + t
//   out = sum_j softmax(s)_j v8_j vs[page_j, g]
// Rows t >= n_b are zeros.
#pragma once

#include "paged_sm100.cuh"

namespace du {

struct ExtendPagedParams {
  const void* q;      // [B, Hq, T, D]
  const uint8_t* k8;  // [N, Hkv, block, D]
  const uint8_t* v8;
  const float* ks;    // [N, Hkv]
  const float* vs;
  const int* table;   // [B, width]
  const int* past;    // [B]
  const int* lens;    // [B]
  const void* cos;    // [positions, D/2]
  const void* sin;
  void* out;          // [B, Hq, T, D]
  int max_len;        // tokens that the table's row and the rope tables cover
  int D, bf16;
  int B, Hq, Hkv, G, T, N, width, block;
  float scale_log2;
};

__device__ __forceinline__ float load16(const void* p, long long i, bool bf16) {
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return bf16 ? __uint_as_float(static_cast<uint32_t>(u) << 16) : __half2float(__ushort_as_half(u));
}

// One warp per query row, one key at a time; a lane has the elements lane, lane + 32, ...
__global__ void __launch_bounds__(128) extend_paged_kernel(const ExtendPagedParams p) {
  const int lane = threadIdx.x & 31;
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.T;
  const long long warps = static_cast<long long>(gridDim.x) * 4;
  const int half = p.D / 2;
  griddep_wait();
  for (long long r = (static_cast<long long>(blockIdx.x) * 128 + threadIdx.x) >> 5; r < rows; r += warps) {
    const int t = static_cast<int>(r % p.T);
    const int h = static_cast<int>(r / p.T % p.Hq), b = static_cast<int>(r / p.T / p.Hq), g = h / p.G;
    const int past = p.past[b], len = p.lens[b];
    const bool ok = past >= 0 && len >= past && len <= p.max_len && len - past <= p.T;
    if (!ok && lane == 0 && h == 0 && t == 0) record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(len));
    const int keys = ok && t < len - past ? past + t + 1 : 0;
    float q[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      q[i] = o[i] = 0.f;
      if (d < p.D && keys > 0) {
        const int j = d < half ? d : d - half;
        const float x1 = load16(p.q, r * p.D + j, p.bf16), x2 = load16(p.q, r * p.D + j + half, p.bf16);
        const long long at = static_cast<long long>(keys - 1) * half + j;
        const float c = load16(p.cos, at, p.bf16), s = load16(p.sin, at, p.bf16);
        q[i] = (d < half ? x1 * c - x2 * s : x2 * c + x1 * s) * p.scale_log2;
      }
    }
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < keys; ++j) {
      const int id = p.table[static_cast<long long>(b) * p.width + j / p.block];
      const bool good = static_cast<unsigned>(id) < static_cast<unsigned>(p.N);
      if (!good && lane == 0) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(id));
      const long long cell = good ? static_cast<long long>(id) * p.Hkv + g : 0;
      const long long at = (cell * p.block + j % p.block) * p.D;
      const float ks = good ? p.ks[cell] : __int_as_float(0x7fc00000), vs = p.vs[cell];
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < p.D) s = fmaf(q[i], e4m3x2_widen(p.k8[at + lane + 32 * i]).x, s);
#pragma unroll
      for (int w = 16; w >= 1; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= ks;
      const float m_new = fmaxf(m, s);
      const float scale = m == m_new ? 1.f : exp2f(m - m_new), w = exp2f(s - m_new);
      l = l * scale + w;
      m = m_new;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < p.D) o[i] = fmaf(w, e4m3x2_widen(p.v8[at + lane + 32 * i]).x * vs, o[i] * scale);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d >= p.D) continue;
      const float x = keys > 0 ? o[i] / l : 0.f;
      if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[r * p.D + d] = __float2bfloat16(x);
      else static_cast<__half*>(p.out)[r * p.D + d] = __float2half(x);
    }
  }
}

}  // namespace du
