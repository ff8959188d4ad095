// Paged KV cache held in 8 bits (e4m3, one fp32 scale per block of tokens and KV head): the
// block tables and slot maps of a step, and the writer of the new tokens' keys and values. The
// attention that reads the cache is in decode_paged_sm100.cuh.
#pragma once

#include "du_ptx.cuh"

namespace du {

// ---------------------------------------------------------------------------------------------
// e4m3 helpers
// ---------------------------------------------------------------------------------------------
// Two fp32 values to a packed e4m3 pair (a in the low byte), nearest-even, saturating at 448.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// A packed pair of 16-bit values as two fp32 values (bf16: one shift and one mask).
template <bool BF16>
__device__ __forceinline__ float2 split2(uint32_t w) {
  return f2_split(widen2<BF16>(w));
}

// Four fp32 values to packed e4m3, a in the lowest byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// A packed e4m3 pair widened to fp32 (exact).
__device__ __forceinline__ float2 e4m3x2_widen(uint32_t p) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(p)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// x / y for a quotient of at most 2^21 (x >= 0, y > 0): a float estimate, off by one at most, and a
// step. (Chunks of a request, which the host keeps at 2^20, units of one, requests, CTAs.)
__device__ __forceinline__ int small_div(int x, int y) {
  int q = static_cast<int>(__fdividef(static_cast<float>(x), static_cast<float>(y)));
  const int r = x - q * y;
  return q + (r >= y) - (r < 0);
}

// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Brings a word into L1 and waits for nothing.
__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("{\n\t.reg .b32 t;\n\tld.global.b32 t, [%0];\n\t}\n" ::"l"(p));
}

// ---------------------------------------------------------------------------------------------
// Block tables and slot maps
// ---------------------------------------------------------------------------------------------
struct PagedTablesParams {
  int* table;           // [B, width], updated in place
  const int* old_lens;  // [B] tokens cached
  const int* new_lens;  // [B] tokens wanted
  int* ring;            // [N] free block ids: a ring, taken at its head, given back at its tail
  const int* state;     // {head, count} of the ring
  int* slots;           // [B, T]
  int* lens_out;        // [B]
  int* state_out;       // {head, count}
  int B, width, N, block, T;
};

constexpr int PAGED_TABLES_THREADS = 512;
constexpr int PAGED_MAX_BATCH = 8192;  // two prefix sums per request in shared memory (64 KB)

// A request's pages before and after, as asked for. A request whose lengths are out of range
// asks for what it has.
struct PagedAsk {
  int old_len, new_len, old_pages, new_pages;
  bool bad;
};
__device__ __forceinline__ PagedAsk paged_ask(const PagedTablesParams& p, int b, bool ring_ok) {
  PagedAsk a;
  a.old_len = p.old_lens[b];
  a.new_len = p.new_lens[b];
  const int cap = p.width * p.block;  // (the host checks that it fits)
  a.bad = a.old_len < 0 || a.old_len > cap || a.new_len < 0 || a.new_len > cap ||
          a.new_len - a.old_len > p.T;
  if (a.bad || !ring_ok) a.new_len = a.old_len;
  const int o = min(max(a.old_len, 0), cap), n = min(max(a.new_len, 0), cap);
  a.old_pages = (o + p.block - 1) / p.block;
  a.new_pages = (n + p.block - 1) / p.block;
  return a;
}

// Last index with off[i] <= x (off is non-decreasing, off[0] = 0): among requests with equal
// offsets that is the one that holds element x, since those before it hold none.
__device__ __forceinline__ int paged_owner(const int* off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Block tables and slot maps of a step from the requests' lengths, in one launch.
//
// pages(n) = ceil(n / block). Request b needs need_b = max(0, pages(new_b) - pages(old_b)) more
// blocks and gives back max(0, pages(old_b) - pages(new_b)); it is served if need_b = 0 or the
// needs of requests 0..b sum to at most the free blocks. Taken entries, in (request, page) order,
// get the ring's blocks from its head on; given-back entries go behind its tail. The two ranges
// of the ring never meet (free + given back <= N), entries that are read as held blocks lie
// before every entry that is written, and a slot's new block is read from the ring, so no CTA
// waits for another: every CTA repeats the scan of the lengths (two loads per request, L2) and
// takes a share of the entries and slots. Bound by latency: the loads of the lengths, the scan,
// the loads of ring or table. Measured (B200, calls in a CUDA graph): 64 requests of one new token
// 3.6 us, 16 of 4096 each 6.1 us, 512 of up to 257 each 6.2 us.
__global__ void __launch_bounds__(PAGED_TABLES_THREADS) paged_tables_kernel(const PagedTablesParams p) {
  extern __shared__ int sm_off[];  // take[B], give[B]: exclusive prefix sums
  __shared__ int warp_sum[2][PAGED_TABLES_THREADS / 32];
  __shared__ int served_sum[PAGED_TABLES_THREADS / 32];
  int* take = sm_off;
  int* give = sm_off + p.B;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int NW = PAGED_TABLES_THREADS / 32;
  griddep_wait();

  const int head = p.state[0], count = p.state[1];
  bool ring_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;

  int carry_t = 0, carry_g = 0, taken_max = 0;
  for (int pass = 0; pass < 2; ++pass) {
    carry_t = carry_g = taken_max = 0;
    for (int b0 = 0; b0 < p.B; b0 += PAGED_TABLES_THREADS) {
      const int b = b0 + tid;
      int need = 0, back = 0;
      if (b < p.B) {
        const PagedAsk a = paged_ask(p, b, ring_ok);
        need = max(0, a.new_pages - a.old_pages);
        back = max(0, a.old_pages - a.new_pages);
        if (a.bad && blockIdx.x == 0 && pass == 0)
          record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(p.new_lens[b]));
      }
      int it = need, ig = back;  // inclusive scans
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, it, o), g = __shfl_up_sync(0xffffffffu, ig, o);
        if (lane >= o) {
          it += t;
          ig += g;
        }
      }
      if (lane == 31) {
        warp_sum[0][warp] = it;
        warp_sum[1][warp] = ig;
      }
      __syncthreads();
      int bt = carry_t, bg = carry_g, tt = 0, tg = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const int xt = warp_sum[0][w], xg = warp_sum[1][w];
        if (w < warp) {
          bt += xt;
          bg += xg;
        }
        tt += xt;
        tg += xg;
      }
      it += bt;
      ig += bg;
      if (b < p.B) {
        take[b] = it - need;
        give[b] = ig - back;
        if (need > 0 && it <= count) taken_max = max(taken_max, it);
      }
      carry_t += tt;
      carry_g += tg;
      __syncthreads();
    }
    // More given back than the ring has room for: the ring's state is not the tables'. Nothing
    // changes hands then (scanned once more with every request kept as it is).
    if (!ring_ok || static_cast<long long>(count) + carry_g <= p.N) break;
    ring_ok = false;
  }
  if (!ring_ok && blockIdx.x == 0 && tid == 0)
    record_error(7u, static_cast<unsigned>(head), static_cast<unsigned>(count));
  // Blocks taken: the largest prefix sum of needs that the free blocks cover.
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) taken_max = max(taken_max, __shfl_xor_sync(0xffffffffu, taken_max, o));
  if (lane == 0) served_sum[warp] = taken_max;
  __syncthreads();
  int taken = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) taken = max(taken, served_sum[w]);
  const int given = carry_g;

  const long long first = static_cast<long long>(blockIdx.x) * PAGED_TABLES_THREADS + tid;
  const long long step = static_cast<long long>(gridDim.x) * PAGED_TABLES_THREADS;
  auto ring_at = [&](long long i) { return static_cast<int>((static_cast<long long>(head) + i) % p.N); };
  for (long long a = first; a < taken; a += step) {
    const int b = paged_owner(take, p.B, static_cast<int>(a));
    const PagedAsk q = paged_ask(p, b, ring_ok);
    p.table[static_cast<long long>(b) * p.width + q.old_pages + (a - take[b])] = p.ring[ring_at(a)];
  }
  for (long long f = first; f < given; f += step) {
    const int b = paged_owner(give, p.B, static_cast<int>(f));
    const PagedAsk q = paged_ask(p, b, ring_ok);
    const int id = p.table[static_cast<long long>(b) * p.width + q.new_pages + (f - give[b])];
    // (it keeps its place in the ring: the ranks of the others are known before any entry is read)
    if (id < 0 || id >= p.N) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(id));
    p.ring[ring_at(count + f)] = id;
  }
  const long long n_slots = static_cast<long long>(p.B) * p.T;
  for (long long i = first; i < n_slots; i += step) {
    const int b = static_cast<int>(i / p.T), t = static_cast<int>(i - static_cast<long long>(b) * p.T);
    const PagedAsk q = paged_ask(p, b, ring_ok);
    const int need = q.new_pages - q.old_pages;
    const bool served = need <= 0 || take[b] + need <= count;
    int slot = -1;
    // (a bad request asks for no more than it has: no new token)
    if (served && t < q.new_len - q.old_len) {
      const int pos = q.old_len + t, page = pos / p.block;
      const int id = page < q.old_pages ? p.table[static_cast<long long>(b) * p.width + page]
                                        : p.ring[ring_at(take[b] + page - q.old_pages)];
      // an id outside the cache gives no slot (the block table was damaged)
      if (id >= 0 && id < p.N) slot = id * p.block + (pos - page * p.block);
      else record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(id));
    }
    p.slots[i] = slot;
  }
  if (blockIdx.x == 0) {
    for (int b = tid; b < p.B; b += PAGED_TABLES_THREADS) {
      const PagedAsk q = paged_ask(p, b, ring_ok);
      const int need = q.new_pages - q.old_pages;
      p.lens_out[b] = (need <= 0 || take[b] + need <= count) ? q.new_len : q.old_len;
    }
    if (tid == 0) {
      p.state_out[0] = ring_ok ? ring_at(taken) : head;
      p.state_out[1] = ring_ok ? count - taken + given : count;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Writer
// ---------------------------------------------------------------------------------------------
struct PagedWriteParams {
  const void* k;     // [B, Hkv, T, D] 16-bit, not rotated
  const void* v;     // [B, Hkv, T, D]
  uint8_t* k8;       // [N, Hkv, block, D] e4m3
  uint8_t* v8;
  float* ks;         // [N, Hkv]
  float* vs;
  const int* slots;  // [B, T]: block * block_size + row, -1: no token
  const int* past;   // [B]: position of the request's first new token
  const void* cos;   // [positions, D/2]
  const void* sin;
  long long positions;
  int B, Hkv, T, N, block, pages;  // pages: blocks that one request's T tokens can touch
  int items;         // B pages Hkv
  int d_log2, block_log2;  // head_dim = 2^d_log2, block = 2^block_log2
};

// a b + c rounded to odd: the exact value where it has 24 bits, else the one of its two neighbours
// whose last bit is set. Rounding that to e4m3 gives what rounding the exact value would (no double
// rounding), and no inexact value lands on the border of a scale. The neighbours come from
// rounding down and up: they differ in their last bit unless the value is exact.
__device__ __forceinline__ float fma_odd(float a, float b, float c) {
  const float lo = __fmaf_rd(a, b, c), hi = __fmaf_ru(a, b, c);
  return (__float_as_uint(lo) & 1u) ? lo : hi;
}

// The smallest power of two of at least 2^-64 whose 448-fold covers amax (its bits given); NaN
// when amax is not finite.
__device__ __forceinline__ float paged_unit(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __int_as_float(0x7fc00000);
  // amax = f 2^x with f in [1, 2): 448 = 1.75 2^8
  const int x = static_cast<int>(amax_bits >> 23) - 127;
  const int e = max((amax_bits & 0x7fffffu) <= 0x600000u ? x - 8 : x - 7, -64);
  return __int_as_float((e + 127) << 23);
}

// Resident warps per SM that the writer's registers are kept to, by the chunk pairs per thread.
constexpr int paged_write_warps(int pairs) { return pairs == 4 ? 16 : (pairs == 2 ? 24 : 32); }

// Quantises the new tokens of a call into the cache: keys rotated at their positions, one scale
// per (block, KV head) and per cache.
//
// A work item is (request, block that its tokens touch, KV head), its keys and then its values; WPI
// warps take it, a thread NP (at most four) pairs of 16-byte chunks i, i + D/2 of a row, which is what a
// rotation pairs up, held in registers from the load to the store. The largest magnitude of the
// item's rows gives the scale: the smallest power of two with amax <= 448 scale, or the block's
// present scale where that is larger and the block holds rows already. Products of two 16-bit values
// are exact in fp32, their sum is rounded to odd and the scale is a power of two, so each byte is
// the e4m3 value nearest to the exact quotient. Where a block's scale grows, its present rows are
// scaled down and rounded again; that is exact but for what falls below the format's normal range.
// A block with a value that is not finite gets the scale NaN, which every attention over it then
// returns.
//
// Bound by the issue slots in prompts (56 % of them), then by HBM (2 bytes read and 1 written per
// value): about 10 instructions per key value and 4 per value, besides some 400 per item and warp
// for addresses and slots. By the chain of loads (length, rows and slots, scale) for single tokens.
// Measured (B200, calls in a CUDA graph): 4 prompts of up to 8192 tokens, 8 KV heads of 128, blocks
// of 16 33.8 us, 4.9 TB/s; 5 chunks of up to 777, 32 heads of 64 11.7 us, 3.3 TB/s; 64 single
// tokens, 8 heads of 128 2.5 us. With four chunk pairs for every item the last one took 4.5 us.
template <bool BF16, int WPI, int NP>
__device__ __forceinline__ void paged_write_item(const PagedWriteParams& p, int b, int pg, int h, uint32_t (*warp_max)[WPI]) {
  constexpr int NT = 32 * WPI;  // threads per item
  const int lane_i = threadIdx.x % NT;  // thread within the item
  const int D = 1 << p.d_log2;
  const int past = p.past[b];
  const int row0 = past >= 0 ? past & (p.block - 1) : 0;  // row of the request's first new token
  const int t0 = pg == 0 ? 0 : (pg << p.block_log2) - row0;
  if (t0 >= p.T) return;
  const int r0 = pg == 0 ? row0 : 0;  // the block's first row that this call writes
  const int n = min(p.T - t0, p.block - r0);
  const int* slot_row = p.slots + static_cast<long long>(b) * p.T + t0;
  // This thread's chunk pairs: chunk c of rows r, r + dr, ... (NT threads hold whole rows).
  const int pairs_log2 = p.d_log2 - 4;
  const int r = lane_i >> pairs_log2, c = lane_i & ((1 << pairs_log2) - 1), dr = NT >> pairs_log2;
  const long long x0 = ((static_cast<long long>(b) * p.Hkv + h) * p.T + t0 + r) * (2 * D) + c * 16;
  const uint8_t* kx = static_cast<const uint8_t*>(p.k) + x0;
  const uint8_t* vx = static_cast<const uint8_t*>(p.v) + x0;
  // Rows that the tables reach (of values too: a token is written whole or not).
  const int reach = past < 0 ? 0 : static_cast<int>(max(0LL, min(static_cast<long long>(n), p.positions - past - t0)));
  const long long pos0 = static_cast<long long>(past) + t0 + r;
  const uint8_t* cosp = static_cast<const uint8_t*>(p.cos) + pos0 * D + c * 16;
  const uint8_t* sinp = static_cast<const uint8_t*>(p.sin) + pos0 * D + c * 16;
  // Everything whose address is known goes out at once: rows, slots and the rows of the tables. A
  // row beyond the last is the last again, which changes no magnitude. (In prompts, where requests'
  // padding makes whole blocks without tokens, those are left first.)
  uint4 xa[NP], xb[NP], cv[NP], sv[NP], va[NP], vb[NP];
  int slots[NP];
  const int slot0 = slot_row[0];
  int given = -1;  // a slot of this thread's rows
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = r + i * dr;
    slots[i] = row < n ? slot_row[row] : -1;
    given = max(given, slots[i]);
  }
  if (reach == 0 || (p.T > p.block && slot0 < 0)) {
    if (given >= 0) {  // beyond the tables, or behind a row without a token
      if (reach == 0) record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(past < 0 ? past : past + t0));
      else record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(given));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int step = min(r + i * dr, reach - 1) - r;
    xa[i] = ldg_stream_v4(kx + step * (2 * D));
    xb[i] = ldg_stream_v4(kx + step * (2 * D) + D);
    cv[i] = ldg_v4(cosp + step * D);
    sv[i] = ldg_v4(sinp + step * D);
    va[i] = ldg_stream_v4(vx + step * (2 * D));
    vb[i] = ldg_stream_v4(vx + step * (2 * D) + D);
  }
  if (slot0 < 0) {  // no token here
    if (given >= 0) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(given));
    return;
  }
  const int blk = slot0 >> p.block_log2;
  if (blk >= p.N || (slot0 & (p.block - 1)) != r0) {
    if (lane_i == 0) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(slot0));
    return;
  }
  const long long cell = static_cast<long long>(blk) * p.Hkv + h;
  const float had_k = r0 > 0 ? p.ks[cell] : 0.f, had_v = r0 > 0 ? p.vs[cell] : 0.f;
  unsigned live = 0;  // pairs of rows that hold a token
  int wrong = -1;     // a row whose slot or position is not fit, and its code
  unsigned code = 0;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = r + i * dr;
    const bool on = slots[i] == slot0 + row && row < reach;
    if (slots[i] >= 0 && !on) {
      const bool far = slots[i] == slot0 + row;
      wrong = far ? past + t0 + row : slots[i];
      code = far ? 6u : 7u;
    }
    live |= on ? 1u << i : 0u;
  }
  if (wrong >= 0) record_error(code, static_cast<unsigned>(b), static_cast<unsigned>(wrong));

  // The rows' values y into the block of one cache.
  auto put = [&](float (&y1)[NP][8], float (&y2)[NP][8], float* scale, uint8_t* cells, float had, uint32_t* maxima) {
    float peak = 0.f;  // the largest magnitude (NaN stays)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      float high = peak;
#pragma unroll
      for (int e = 0; e < 8; ++e) high = max3_abs_nan(high, y1[i][e], y2[i][e]);
      peak = (live & (1u << i)) ? high : peak;
    }
    // Bits of the magnitude, NaN above infinity above every number; one more, 0: no row.
    uint32_t top = live ? (__float_as_uint(peak) & 0x7fffffffu) + 1u : 0u;
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (WPI > 1) {
      if ((threadIdx.x & 31) == 0) maxima[threadIdx.x >> 5] = top;
      __syncthreads();  // (and every thread has read the present scales)
#pragma unroll
      for (int w = 0; w < WPI; ++w) top = max(top, maxima[w]);
    }
    if (top == 0) return;  // the item's: nothing is written, the scale neither
    float unit = paged_unit(top - 1);
    if (r0 > 0 && (unit <= had || had != had)) unit = had;  // (a NaN on either side stays)
    if (lane_i == 0) scale[cell] = unit;
    const bool poison = unit != unit;
    const float inv = 1.0f / unit;
    uint8_t* out = cells + cell * p.block * D;
    uint8_t* dst = out + (r0 + r) * D + 8 * c;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (!(live & (1u << i))) continue;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        w[e] = e4m3x4(y1[i][4 * e] * inv, y1[i][4 * e + 1] * inv, y1[i][4 * e + 2] * inv, y1[i][4 * e + 3] * inv);
        w[2 + e] = e4m3x4(y2[i][4 * e] * inv, y2[i][4 * e + 1] * inv, y2[i][4 * e + 2] * inv, y2[i][4 * e + 3] * inv);
      }
      if (poison) w[0] = w[1] = w[2] = w[3] = 0x7f7f7f7fu;
      *reinterpret_cast<uint2*>(dst + i * 16 * NT) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + i * 16 * NT + D / 2) = make_uint2(w[2], w[3]);
    }
    if (r0 > 0 && unit > had) {
      // The present rows under the larger scale.
      const float f = had * inv;
      for (int u = lane_i; u < r0 * (D / 16); u += NT) {
        uint4* q = reinterpret_cast<uint4*>(out) + u;
        const uint4 o = *q;
        uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 lo = e4m3x2_widen(w[e] & 0xffffu), hi = e4m3x2_widen(w[e] >> 16);
          w[e] = e4m3x4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
        }
        *q = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };

  float y1[NP][8], y2[NP][8];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint32_t aw[4] = {xa[i].x, xa[i].y, xa[i].z, xa[i].w}, dw[4] = {xb[i].x, xb[i].y, xb[i].z, xb[i].w};
    const uint32_t cw[4] = {cv[i].x, cv[i].y, cv[i].z, cv[i].w}, sw[4] = {sv[i].x, sv[i].y, sv[i].z, sv[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (products of two 16-bit values are exact)
      const float2 v = split2<BF16>(aw[e]), w = split2<BF16>(dw[e]);
      const float2 cc = split2<BF16>(cw[e]), ss = split2<BF16>(sw[e]);
      y1[i][2 * e] = fma_odd(v.x, cc.x, -__fmul_rn(w.x, ss.x));
      y1[i][2 * e + 1] = fma_odd(v.y, cc.y, -__fmul_rn(w.y, ss.y));
      y2[i][2 * e] = fma_odd(w.x, cc.x, __fmul_rn(v.x, ss.x));
      y2[i][2 * e + 1] = fma_odd(w.y, cc.y, __fmul_rn(v.y, ss.y));
    }
  }
  put(y1, y2, p.ks, p.k8, had_k, warp_max[0]);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint32_t aw[4] = {va[i].x, va[i].y, va[i].z, va[i].w}, dw[4] = {vb[i].x, vb[i].y, vb[i].z, vb[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = split2<BF16>(aw[e]), w = split2<BF16>(dw[e]);
      y1[i][2 * e] = v.x;
      y1[i][2 * e + 1] = v.y;
      y2[i][2 * e] = w.x;
      y2[i][2 * e + 1] = w.y;
    }
  }
  put(y1, y2, p.vs, p.v8, had_v, warp_max[1]);
}

template <bool BF16, int WPI, int NP>
__global__ void __launch_bounds__(WPI == 1 ? 128 : 32 * WPI, paged_write_warps(NP) / (WPI == 1 ? 4 : WPI))
    paged_write_kernel(const PagedWriteParams p) {
  // Warps' maxima of keys and of values: each is written again only after the other one's barrier.
  __shared__ uint32_t warp_max[2][WPI];
  griddep_launch_dependents();
  griddep_wait();
  // A grid of resident CTAs walks the items (short CTAs, one per item, ended faster than new ones
  // came: 13 of 64 warps per SM at any time). With WPI = 1 a warp is an item; else the CTA is one,
  // and its barriers are reached by all or none.
  const int per_request = p.Hkv * p.pages;
  const int stride = static_cast<int>(gridDim.x) * (WPI == 1 ? 4 : 1);
  for (int item = WPI == 1 ? static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x) / 32 : static_cast<int>(blockIdx.x);
       item < p.items; item += stride) {
    const int b = small_div(item, per_request), in = item - b * per_request;
    const int pg = small_div(in, p.Hkv);
    paged_write_item<BF16, WPI, NP>(p, b, pg, in - pg * p.Hkv, warp_max);
  }
}

}  // namespace du
