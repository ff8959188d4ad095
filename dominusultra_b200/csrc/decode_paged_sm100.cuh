// Single-token attention over the paged 8-bit KV cache (layout in paged_sm100.cuh), on tcgen05.
//
// Per request b with n cached tokens (the query's own among them) and query head h of KV head g:
//   q' = R(n - 1) q            s_j = (q' . k8_j) ks[page_j, g] scale       j < n
//   out = sum_j softmax(s)_j v8_j vs[page_j, g]
// The cached keys are rotated already. A request without tokens gives zeros.
//
// The call streams the cache once (1 byte per value) and should run at HBM speed: about 23 bytes
// per clock and SM. Widening each byte on the CUDA cores would take most of their issue slots, so
// the cached bytes go to the tensor cores as they are (kind::f8f6f4, e4m3 x e4m3 -> fp32) and the
// few operands on the other side are carried as sums of e4m3 parts instead, each part what the parts
// before it left, scaled up:
//   query    x = x1 + x2 2^-4 + x3 2^-8,               x1 = e4m3(x), x2 = e4m3(2^4 (x - x1)), ...
//   weight   w = w1 + w2 2^-5 + w3 2^-10 + w4 2^-15    (w rounded to fp16 first)
// A query's part holds 4 significant bits, so three carry 12: half a step of 2^-12, as fp16 operands
// would. A weight is at most 2^8, where a part leaves at most 2^3: the next one can be scaled by 2^5.
// Three parts then hold any fp16 weight of at least 2^-9 and the fourth the smaller ones down to fp16's
// last step, 2^-24 (e4m3's last step is 2^-9), so the four are the fp16 weight exactly. The parts are
// rows of their own in tiles that are mostly empty otherwise, so they cost no tensor time:
//   S^T = K8 Q^T     M = 128 keys of a chunk, N = 16 or 32 (three parts of the unit's heads),
//                    K = head_dim. A = the K tile as TMA left it, B = the query parts.
//   O  += P V8       M = 64 or 128, N = head_dim, K = 128 keys. A = P, B = the V tile as TMA left
//                    it (MN-major). Row (M/4) w + t HPU + h: part t of head h's weights at warp w's
//                    keys, which TMEM lane 32 w + t HPU + h holds.
// One key per TMEM lane, so the softmax is one thread per key, and each of its four warps keeps a
// reference maximum, a sum and rows of O of its own over its 32 keys of every chunk: no
// reduction across warps per chunk. The value scale joins the weight before it is split: with
// u_j = s_j + log2 vs_j (log2 domain) the carried weight is 2^(u_j - m) = w_j vs_j. The sum takes
// 2^(u_j - m - log2 vs_j), an exponential of its own: value scales may be 2^190 apart, and a key whose
// carried weight is nothing beside another's can have all of the softmax's. (2^24 times that: without the
// factor its largest term lies between 2^-121 and 2^72, too near to the smallest float; with it 2^27 terms
// stay below 2^123.) m moves only when some u exceeds it by 8 (then to 7 below that
// maximum), so the weights stay within 2^8 and the largest one of a warp is at least 2^7. Half a step of
// the smallest weights is 2^-25 then, 2^-32 of the largest: behind a key that takes nearly all of the
// weight and has values of zero, a long tail keeps its part. (With three parts, a factor of 2^4
// between them and the largest weight at 2^4 the floor was 2^-22, and a tail of that size 26 % off.)
//
// Work: the requests' chunks of 128 keys, unit by unit (unit: request, KV head, group of up to
// HPU query heads), cut into equal ranges, one per CTA of a persistent grid. Lengths are read on
// the device; every CTA repeats the sum over them. A unit within one CTA is written at once; the
// fragments of others leave fp32 partials, and the CTA that leaves the last one joins them.
//
// Warps: 0-3 softmax, combine and output; 4 TMA of K, and the scales; 7 TMA of V (a block of 16 tokens
// is a copy of 2 KB, and one warp issues a copy in about 100 clocks: half an SM's share of the
// bandwidth); 5 TMEM and MMA; 6 walks the fragments and prepares their query parts, ahead of the
// others. Every wait is bounded.
//
// Measured (B200, calls in a CUDA graph): 4 requests of 131072 tokens, 32 heads on 8 of 128 162-165 us, 6.5
// TB/s, the rate of a copy; 16 of up to 20001, 64 on 8 of 128 66-68 us, 5.2 TB/s; 64 of up to 4096, 32 on
// 8 of 128, blocks of 16 52.4 us, 5.2 TB/s; one of 32768, the same heads 21.8 us; 8 of 2048, 32 on 32 of 64
// 17.6 us; 16 of 16384, 4 on 2 of 256 50.5 us, 5.3 TB/s; one of 100, 8 heads of 64 5.7 us. Long contexts are
// bound by HBM; the others by the start (length, table and first copies: some 4500 clocks before the first
// byte is asked for) and by the ends of fragments.
#pragma once

#include <float.h>

#include "paged_sm100.cuh"

namespace du {

struct DecodePagedParams {
  const void* q;        // [B, Hq, D]
  const float* ks;      // [N, Hkv]
  const float* vs;
  const int* table;     // [B, width]
  const int* lens;      // [B]
  const void* cos;      // [positions, D/2]
  const void* sin;
  void* out;            // [B, Hq, D]
  int* cnt;             // [gridDim.x] tickets, zero between calls
  float* part;          // [2 gridDim.x][HPU][D] partial outs, then [2 gridDim.x][HPU] log2 of their sums
  int max_len;          // tokens that the table's row and the rope tables cover
  int D, bf16;
  int B, Hq, Hkv, G, N, width;
  int block, block_log2;
  int n_gchunk, heads;  // groups of `heads` query heads per KV head (the last may hold fewer)
  float scale_log2;
};

// Chunks per CTA that whole pieces of units may cost over equal ranges of chunks: a CTA whose range
// straddles two units combines twice, about three chunks' time.
constexpr int DECODE_PAGED_PIECE_SLACK = 3;
// What a warp's reference lies below its maximum when it moves, in octaves (see above).
constexpr float DECODE_PAGED_BELOW = 7.0f;
// The CTA that joins a unit holds a weight per fragment and head where P is otherwise.
constexpr int DECODE_PAGED_MAX_CTAS = 12 * 36;
__device__ float g_du_paged_nan = __builtin_nanf("");  // the scale of a block that does not exist

// cp.async of 4 and of 16 bytes, their groups, and an arrival on `bar` once this thread's earlier
// cp.async have landed.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// D[tmem] (+)= A[smem] * B[smem], e4m3 operands, fp32 accumulate, one CTA.
__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The four e4m3 parts of two weights (packed fp16, 0 <= value <= 256), each part packed as a pair.
__device__ __forceinline__ void e4m3_parts2(uint32_t x, uint32_t (&t)[4]) {
  uint32_t r = x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t e;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(e) : "r"(r));
    t[i] = e;
    if (i < 3) {
      uint32_t f;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f) : "h"(e));
      const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&f));
      const __half2 s = __hmul2(d, __float2half2_rn(32.0f));  // exact: d has at most 7 bits, and is at most 8
      r = *reinterpret_cast<const uint32_t*>(&s);
    }
  }
}

template <int DP_, int HPU_>
struct DecodePagedShape {
  static constexpr int DP = DP_;    // head_dim (32 for head_dim 16: the upper half is zero)
  static constexpr int HPU = HPU_;  // query heads per unit
  static constexpr int NQ = 3 * HPU <= 16 ? 16 : 32;  // rows of the query tile
  static constexpr int CK = 128;    // keys per chunk
  static constexpr int SPAN = DP < 128 ? DP : 128;    // bytes per row of a swizzled block
  static constexpr int NBLK = DP / SPAN;
  static constexpr int TILE = CK * DP;
  // Two CTAs per SM where their tiles allow: one's softmax, fragment ends and start overlap the
  // other's copies.
  static constexpr int CTAS = DP <= 128 ? 2 : 1;
  static constexpr int NPB = DP == 128 && HPU == 8 ? 1 : 2;  // P buffers
  static constexpr int PM = HPU <= 4 ? 64 : 128;      // rows of P (M of P V): 16 or 32 per warp
  static constexpr int P_BYTES = CK * PM;             // [key][PM rows] bytes, swizzled
  static constexpr int Q_BYTES = ((NQ * DP + 1023) / 1024) * 1024;
  // Rows of O are combined where P is, CB columns at a time (and P's zeros put back): 4 warps x
  // 4 HPU rows of CB floats, a row's 16-byte parts in an order that the row's number gives.
  static constexpr int CB = DP < 64 ? DP : (DP == 128 && HPU == 8 ? 32 : 64);
  static constexpr int ML_BYTES = ((8 * HPU * 4) + 127) / 128 * 128;  // maxima and sums of the warps
  static constexpr int RAW_BYTES = (HPU + 1) * DP * 2;  // a unit's query rows and its cos and sin row
  static constexpr int FIXED = NPB * P_BYTES + 2 * Q_BYTES + ML_BYTES + 2 * RAW_BYTES + 2560;
  static constexpr int BUDGET = CTAS == 2 ? 113 * 1024 : 226 * 1024;
  static constexpr int TILES = (BUDGET - FIXED) / TILE;
  static constexpr int NV = TILES / 2 > 8 ? 8 : TILES / 2;            // stages of V
  static constexpr int NK = TILES - NV > 8 ? 8 : TILES - NV;          // stages of K and scales
  static constexpr int OFF_V = NK * TILE;
  static constexpr int OFF_P = OFF_V + NV * TILE;
  static constexpr int OFF_Q = OFF_P + NPB * P_BYTES;
  static constexpr int OFF_ML = OFF_Q + 2 * Q_BYTES;
  static constexpr int OFF_RAW = OFF_ML + ML_BYTES;
  static constexpr int OFF_SC = OFF_RAW + 2 * RAW_BYTES;  // [NK][2][8] scales of a chunk's blocks
  static constexpr int NF = 4;                        // fragment entries in flight
  static constexpr int OFF_FRAG = OFF_SC + NK * 64;   // [NF] entries of 16 words
  static constexpr int OFF_OWED = OFF_FRAG + NF * 64; // [2] entries of units to join
  static constexpr int OFF_QS = OFF_OWED + 2 * 64;    // [2][HPU] score factor of each head
  static constexpr int OFF_BAR = OFF_QS + 2 * 32;
  static constexpr int B_KFULL = 0, B_KEMPTY = NK, B_VFULL = 2 * NK, B_VEMPTY = 2 * NK + NV,
                       B_QFULL = 2 * NK + 2 * NV, B_QEMPTY = B_QFULL + 2, B_SFULL = B_QFULL + 4,
                       B_SEMPTY = B_QFULL + 6, B_PFULL = B_QFULL + 8, B_PDONE = B_QFULL + 10,
                       B_MRG = B_QFULL + 12, B_DRAIN = B_QFULL + 13, B_FREE = B_QFULL + 14,
                       B_ML = B_QFULL + 15, B_FFULL = B_QFULL + 16,
                       B_FEMPTY = B_FFULL + NF;
  static constexpr int N_BAR = B_FEMPTY + NF;
  static constexpr int OFF_MISC = OFF_BAR + 8 * N_BAR;  // 16 words
  static constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
  static constexpr int TM_S = 0;           // S^T: two buffers of NQ columns
  static constexpr int TM_O = 64;          // O: DP columns
  static constexpr int TMEM_COLS = TM_O + DP <= 128 ? 128 : (TM_O + DP <= 256 ? 256 : 512);
  static constexpr int NTHREADS = 256;
  // Chunks that a unit's beginning is charged with (measured with 2, 3, 4 and four heads or fewer: 64
  // requests of up to 4096, 32 on 8 heads of 128 51.5, 51.9, 52.4 us; 48 of up to 3000, 16 heads of 64
  // 35.7, 35.1, 36.2 us. With 3, 4, 5, 6 and eight heads: 16 of up to 20001, 64 on 8 heads of 128 66.9,
  // 66.3, 66.9, 67.3 us; 100 of up to 2500, 32 on one of 64 27.1, 27.3, 27.9, 28.2 us).
  static constexpr int PEN = HPU == 8 ? 4 : 3;
  static_assert(4 * HPU <= PM / 4, "a warp's rows of P");
  static_assert(16 * HPU * CB * 4 <= NPB * P_BYTES, "rows of O where P is");
  static_assert(HPU * DECODE_PAGED_MAX_CTAS * 4 <= NPB * P_BYTES, "weights of a unit's fragments where P is");
  static_assert(NV >= 2 && NK >= 2, "at least two stages");
  static_assert(SMEM_BYTES <= (CTAS == 2 ? 115712 : 232448), "shared memory budget");
  static_assert(OFF_SC % 16 == 0 && OFF_BAR % 8 == 0, "alignment");
};

// This CTA's share of the flattened chunks, found by one warp. The host refuses batches whose block
// tables could hold 2^31 chunks, so chunk numbers are ints.
//
// Two plans. pieces > 0: every unit is cut into equal pieces, as many as give no CTA more than one,
// and this CTA has piece `cur` of request b's units (numbered through them), if cur < hi. Else the
// CTA has the chunks [cur, hi), which may begin and end inside a unit; request b holds `cur` and
// starts at chunk `base`; `per` chunks per CTA. There a unit's chunks are preceded by PEN positions
// that hold none: the price, in chunks, of beginning a fragment and combining its rows, so that CTAs
// with many short units get fewer chunks.
struct PagedStart {
  int cur, hi, per;
  int b, base;
  int pieces;
};

// One fragment, as warp 6 leaves it for the other warps (16 words).
struct PagedFrag {
  int kind;       // 1 a fragment, 0 the end
  int b, h0, nh;  // request, first query head, heads
  int chunks;     // 0: a request without tokens
  int keys;       // keys of the fragment
  int nf, c0;     // fragments of the unit, CTA of the first
  int slot;       // partial slot when nf > 1
  int kvh, kbeg;  // KV head, first token
  int len;        // the request's tokens
  int pad[4];
};

// Walks a CTA's share fragment by fragment.
template <int PEN>
struct PagedWalk {
  int cur, hi, per, base, b, pieces;
  __device__ __forceinline__ void init(const PagedStart& s) {
    cur = s.cur;
    hi = s.hi;
    per = s.per;
    base = s.base;
    b = s.b;
    pieces = s.pieces;
  }
  __device__ __forceinline__ static int tokens(const DecodePagedParams& p, int b) {
    const int n = p.lens[b];
    return static_cast<unsigned>(n) > static_cast<unsigned>(p.max_len) ? 0 : n;
  }
  __device__ __forceinline__ static int chunks(int n) { return n > 128 ? (n + 127) >> 7 : 1; }
  // The CTA's share (a whole warp; `lane` its lane).
  __device__ __forceinline__ static PagedStart find(const DecodePagedParams& p, int lane) {
    PagedStart st;
    const int ups = p.Hkv * p.n_gchunk;
    const int grid = static_cast<int>(gridDim.x), c = static_cast<int>(blockIdx.x);
    // The first 32 requests' chunks stay in a register: most batches are no larger.
    const int len0 = lane < p.B ? p.lens[lane] : 0;
    const int nc0 = chunks(static_cast<unsigned>(len0) > static_cast<unsigned>(p.max_len) ? 0 : len0);
    auto chunks_of = [&](int b) { return b < 32 ? nc0 : chunks(tokens(p, b)); };
    int total = lane < p.B ? nc0 : 0;
#pragma unroll 4
    for (int b = 32 + lane; b < p.B; b += 32) total += chunks(tokens(p, b));
    total = static_cast<int>(__reduce_add_sync(0xffffffffu, total));
    // Pieces: with at most x chunks each, the units of request b make ups ceil(chunks_b / x) of
    // them. x = per .. per + 3 are tried; beyond that, fragments of equal ranges cost less.
    bool cut = false;
    int x = 0;
    if (p.B * static_cast<long long>(ups) <= grid) {
      const int per = small_div(total * ups + grid - 1, grid);
#pragma unroll 1
      for (x = per; x <= per + DECODE_PAGED_PIECE_SLACK && !cut; ++x) {
        int sum = 0;
#pragma unroll 1
        for (int b = lane; b < p.B; b += 32) sum += small_div(chunks_of(b) + x - 1, x);
        cut = static_cast<int>(__reduce_add_sync(0xffffffffu, sum)) * ups <= grid;
      }
      --x;  // (the one that was tried last)
    }
    int cur, hi;
    if (cut) {
      cur = c;
      hi = c + 1;
    } else {
      total = (total + p.B * PEN) * ups;  // (the host keeps total + gridDim.x below 2^31)
      x = (total + grid - 1) / grid;  // (may pass what small_div takes)
      cur = static_cast<int>(min(static_cast<long long>(x) * c, static_cast<long long>(total)));
      hi = min(total - cur, x) + cur;
    }
    st.per = x;
    st.cur = st.hi = st.b = st.base = st.pieces = 0;  // no share
    // The request that holds `cur`.
    int before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.B && cur < hi; b0 += 32) {
      const int b = b0 + lane;
      int k = 0;
      if (b < p.B) {
        const int nc = chunks_of(b);
        k = cut ? small_div(nc + x - 1, x) : nc + PEN;
      }
      int in = k;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, cur < before + in * ups);
      if (hit) {
        const int l = __ffs(static_cast<int>(hit)) - 1;
        k = __shfl_sync(0xffffffffu, k, l);
        in = __shfl_sync(0xffffffffu, in, l);
        st.b = b0 + l;
        st.base = before + (in - k) * ups;
        st.cur = cut ? cur - st.base : cur;
        st.hi = cut ? k * ups : hi;
        st.pieces = cut ? k : 0;
        break;
      }
      before += __shfl_sync(0xffffffffu, in, 31) * ups;
    }
    return st;
  }
  __device__ __forceinline__ bool next(const DecodePagedParams& p, PagedFrag& f) {
    int n, nc, unit, j0, j1;
    if (pieces > 0) {
      if (cur >= hi) return false;
      n = tokens(p, b);
      nc = chunks(n);
      unit = small_div(cur, pieces);
      const int piece = cur - unit * pieces;
      const int q = small_div(nc, pieces), r = nc - q * pieces;  // the first r pieces hold a chunk more
      j0 = piece * q + min(piece, r);
      j1 = j0 + q + (piece < r);
      f.c0 = static_cast<int>(blockIdx.x) - piece;
      f.nf = pieces;
      cur = hi;
    } else {
      const int ups = p.Hkv * p.n_gchunk;
      do {
        if (cur >= hi) return false;
        n = tokens(p, b);
        nc = chunks(n);
        const int span = nc + PEN;
        if (cur - base >= span * ups) {
          base += span * ups;
          ++b;
          j1 = 0;
          continue;
        }
        unit = small_div(cur - base, span);
        const int ub = base + unit * span + PEN;  // the unit's first chunk
        const int e = min(hi, ub + nc);
        j0 = max(cur - ub, 0);
        j1 = e - ub;
        f.c0 = small_div(ub, per);
        f.nf = small_div(ub + nc - 1, per) - f.c0 + 1;
        cur = e;
      } while (j1 <= 0);  // (a range that ends before the unit's first chunk)
    }
    const int kvh = p.n_gchunk == 1 ? unit : small_div(unit, p.n_gchunk);
    const int gch = unit - kvh * p.n_gchunk;
    f.kind = 1;
    f.b = b;
    f.h0 = kvh * p.G + gch * p.heads;
    f.nh = min(p.heads, p.G - gch * p.heads);
    f.kvh = kvh;
    f.kbeg = j0 << 7;
    f.len = n;
    f.keys = min(n, j1 << 7) - f.kbeg;
    f.chunks = f.keys > 0 ? j1 - j0 : 0;
    f.slot = 2 * static_cast<int>(blockIdx.x) + (j0 > 0 ? 0 : 1);
    return true;
  }
};

// mbar_wait and mbar_wait_drain with everything but the first look in one place each: the kernel waits
// at some thirty places, and what a fragment runs once is bound by the fetch of its code. The softmax
// warps' waits stay inline at head_dim 128 and 256, where calls make them spill (8 x 32 heads of 2048
// at head_dim 64: 17.9 -> 17.4 us with calls; a mixed batch at head_dim 128: 53.5 -> 55.6 us).
__device__ __noinline__ bool paged_wait_on(uint32_t bar, uint32_t parity, volatile int* failed, unsigned int site) {
  return mbar_wait(bar, parity, failed, site);
}
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, volatile int* failed, unsigned int site) {
  return mbar_try_wait(bar, parity) || paged_wait_on(bar, parity, failed, site);
}
template <int DP>
__device__ __forceinline__ bool softmax_wait(uint32_t bar, uint32_t parity, volatile int* failed, unsigned int site) {
  if constexpr (DP <= 64) return paged_wait(bar, parity, failed, site);
  else return mbar_wait(bar, parity, failed, site);
}
__device__ __noinline__ bool paged_wait_drain(uint32_t bar, uint32_t parity, unsigned int site) {
  return mbar_wait_drain(bar, parity, site);
}

template <int DP, int HPU>
__global__ void __launch_bounds__(DecodePagedShape<DP, HPU>::NTHREADS, DecodePagedShape<DP, HPU>::CTAS)
    decode_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const DecodePagedParams p) {
  using S = DecodePagedShape<DP, HPU>;
  using Walk = PagedWalk<S::PEN>;
  constexpr int CK = S::CK, SPAN = S::SPAN, NK = S::NK, NV = S::NV, NPB = S::NPB, NQ = S::NQ, CB = S::CB;
  constexpr uint32_t SWZ = swizzle_code(SPAN);
  constexpr uint32_t IDESC_QK = idesc_f16(128, NQ, 0, 0, 0, 0);  // (format 0 of kind::f8f6f4: e4m3)
  constexpr uint32_t IDESC_PV = idesc_f16(S::PM, DP, 0, 0, 1, 1);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t sbase = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw_u32);
  auto bar = [&](int i) -> uint32_t { return sbase + S::OFF_BAR + 8u * static_cast<uint32_t>(i); };
  auto KFULL = [&](int s) { return bar(S::B_KFULL + s); };    // K and scales of a stage landed
  auto KEMPTY = [&](int s) { return bar(S::B_KEMPTY + s); };  // QK read K, each softmax warp its scales
  auto VFULL = [&](int s) { return bar(S::B_VFULL + s); };
  auto VEMPTY = [&](int s) { return bar(S::B_VEMPTY + s); };  // PV read V
  auto FFULL = [&](int i) { return bar(S::B_FFULL + i); };    // fragment entry written
  auto FEMPTY = [&](int i) { return bar(S::B_FEMPTY + i); };  // read by each warp but the walker
  auto QFULL = [&](int i) { return bar(S::B_QFULL + i); };    // query parts written
  auto QEMPTY = [&](int i) { return bar(S::B_QEMPTY + i); };  // the fragment's QK done, factors read
  auto SFULL = [&](int i) { return bar(S::B_SFULL + i); };
  auto SEMPTY = [&](int i) { return bar(S::B_SEMPTY + i); };
  auto PFULL = [&](int i) { return bar(S::B_PFULL + i); };
  auto PDONE = [&](int i) { return bar(S::B_PDONE + i); };    // PV of even / odd chunks complete
  // rows of O in the combine area; rows read (and partials stored); a fragment's maxima and sums
  const uint32_t BAR_MRG = bar(S::B_MRG), BAR_FREE = bar(S::B_FREE), BAR_DRAIN = bar(S::B_DRAIN), BAR_ML = bar(S::B_ML);
  uint32_t* misc = reinterpret_cast<uint32_t*>(sgen + S::OFF_MISC);
  volatile int* failed = reinterpret_cast<volatile int*>(misc + 1);
  volatile int* emitted = reinterpret_cast<volatile int*>(misc + 2);  // fragments done with
  volatile int* n_owed = reinterpret_cast<volatile int*>(misc + 3);
  PagedStart* start = reinterpret_cast<PagedStart*>(misc + 4);
  float* mrg = reinterpret_cast<float*>(sgen + S::OFF_P);  // o [4][4 HPU][CB]
  float* mrg_m = reinterpret_cast<float*>(sgen + S::OFF_ML);  // m [4][HPU], l [4][HPU]
  float* mrg_l = mrg_m + 4 * HPU;
  PagedFrag* owed = reinterpret_cast<PagedFrag*>(sgen + S::OFF_OWED);  // units for this CTA to join

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;

  if (warp == 4) {
    for (int i = lane; i < S::N_BAR; i += 32) {
      int n = 1;  // VFULL, VEMPTY, QFULL, SFULL, PDONE, DRAIN, FFULL
      if (i < S::B_KEMPTY) n = 1 + 32;                                              // KFULL
      else if (i < S::B_VFULL) n = 1 + 4;                                           // KEMPTY
      else if (i >= S::B_QEMPTY && i < S::B_SFULL) n = 1 + 4;                       // QEMPTY
      else if ((i >= S::B_SEMPTY && i < S::B_PDONE) || i == S::B_MRG || i == S::B_FREE || i == S::B_ML) n = 4;  // a warp each
      else if (i >= S::B_FEMPTY) n = 7;                                             // FEMPTY
      mbar_init(bar(i), n);
    }
    if (lane == 0) {
      *failed = 0;
      *emitted = 0;
      *n_owed = 0;
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    mbar_fence_init();
  }
  if (warp == 5) {
    // (Only a predecessor whose CTAs all run or have ended lets this grid start early, and none of
    // them takes TMEM after that: the columns taken here starve nothing.)
    tmem_alloc(sbase + S::OFF_MISC, S::TMEM_COLS);
    tmem_relinquish();
  }
  // Launched as a programmatic dependent: what is above runs beside the stream's previous kernel.
  griddep_wait();
  if (warp == 4 || warp == 7) fence_proxy_async_global();  // the written blocks are read by TMA (async proxy)
  if (warp == 5) griddep_launch_dependents();  // (the columns are taken)
  Walk walk;  // warp 6's
  if (warp == 6) {
    const PagedStart st = Walk::find(p, lane);
    if (lane == 0) *start = st;
    walk.init(st);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);

  if (warp == 4 || warp == 7) {
    // ------------------------------------------------------------------ TMA: K and scales, V
    const bool is_k = warp == 4;
    const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
    const uint32_t ring = sbase + (is_k ? 0u : static_cast<uint32_t>(S::OFF_V));
    const int ns = is_k ? NK : NV;
    const int ppc = CK >> p.block_log2;  // blocks of a whole chunk: 1, 2, 4, 8
    int g = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      if (!(ok = __all_sync(0xffffffffu, paged_wait(FFULL(it % S::NF), (it / S::NF) & 1, failed, 800)))) break;
      const PagedFrag f = *reinterpret_cast<const PagedFrag*>(sgen + S::OFF_FRAG + (it % S::NF) * 64);
      __syncwarp();
      if (f.kind == 0) break;
      if (lane == 0) mbar_arrive(FEMPTY(it % S::NF));
      const int* row = p.table + static_cast<long long>(f.b) * p.width + (f.kbeg >> p.block_log2);
      const int pages = (f.keys + p.block - 1) >> p.block_log2;  // of the fragment
      // Lane l holds the ids of blocks at + l and, loaded ahead, at + 32 + l.
      int id = lane < pages ? row[lane] : 0;
      int id_next = lane + 32 < pages ? row[32 + lane] : 0;
      int at = 0;
      for (int j = 0; j < f.chunks; ++j, ++g) {
        const int first = j * ppc;
        if (first >= at + 32) {
          at += 32;
          id = id_next;
          id_next = at + 32 + lane < pages ? row[at + 32 + lane] : 0;
        }
        const int here = min(ppc, pages - first);
        const int s = g % ns;
        const uint32_t st = ring + s * S::TILE;
        const uint32_t full = is_k ? KFULL(s) : VFULL(s);
        const int mine = __shfl_sync(0xffffffffu, id, (first - at) + (lane & 7));
        const bool in = (lane & 7) < here;
        const bool bad = in && (mine < 0 || mine >= p.N);
        if (bad && is_k && lane < 8) record_error(7u, static_cast<unsigned>(f.b), static_cast<unsigned>(mine));
        const long long cell = bad ? static_cast<long long>(p.N) * p.Hkv  // beyond the map: zeros
                                   : static_cast<long long>(mine) * p.Hkv + f.kvh;
        if (g >= ns) ok = paged_wait(is_k ? KEMPTY(s) : VEMPTY(s), ((g / ns) - 1) & 1, failed, 801);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (lane == 0) mbar_expect_tx(full, static_cast<uint32_t>(here << p.block_log2) * DP);
        __syncwarp();
        if (in && lane < 8)
#pragma unroll
          for (int nb = 0; nb < S::NBLK; ++nb)
            tma_load_3d(st + nb * CK * SPAN + (lane << p.block_log2) * SPAN, tm, full, nb * SPAN, 0,
                        static_cast<int>(cell));
        if (is_k) {
          if (in && lane < 16)
            cp_async4(sbase + S::OFF_SC + s * 64 + lane * 4, bad ? &g_du_paged_nan : (lane < 8 ? p.ks : p.vs) + cell);
          cp_async_arrive(full);
        }
      }
    }
    // The last copies land before the CTA may exit.
    for (int j = g > ns ? g - ns : 0; j < g; ++j)
      paged_wait_drain(is_k ? KFULL(j % ns) : VFULL(j % ns), (j / ns) & 1, 802);
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    bool ok = true;
    int g = 0;
    for (int it = 0; ok; ++it) {
      const int qb = it & 1;
      if (!(ok = __all_sync(0xffffffffu, paged_wait(FFULL(it % S::NF), (it / S::NF) & 1, failed, 810)))) break;
      const PagedFrag* f = reinterpret_cast<const PagedFrag*>(sgen + S::OFF_FRAG + (it % S::NF) * 64);
      const int kind = f->kind, n = f->chunks;
      __syncwarp();
      if (kind == 0) break;
      if (leader) mbar_arrive(FEMPTY(it % S::NF));
      __syncwarp();
      // (also without chunks: the queries of entry it are prepared once QEMPTY of entry it - 2 is
      // complete, so this warp's arrivals stay in their phases)
      if (!(ok = __all_sync(0xffffffffu, paged_wait(QFULL(qb), (it >> 1) & 1, failed, 816)))) break;
      if (n == 0) {
        if (leader) mbar_arrive(QEMPTY(qb));
        __syncwarp();
        continue;
      }
      const uint64_t dq = smem_desc(sbase + S::OFF_Q + qb * S::Q_BYTES, 16, 8 * SPAN, SWZ);
      for (int j = 0; j <= n; ++j) {
        if (j < n) {  // S of chunk j
          const int gj = g + j, s = gj % NK;
          ok = paged_wait(KFULL(s), (gj / NK) & 1, failed, 811);
          if (ok && gj >= 2) ok = paged_wait(SEMPTY(gj & 1), ((gj >> 1) - 1) & 1, failed, 812);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          if (leader) {
            const uint64_t dk = smem_desc(sbase + s * S::TILE, 16, 8 * SPAN, SWZ);
#pragma unroll
            for (int kk = 0; kk < DP / 32; ++kk) {
              const uint32_t off_k = ((kk * 32) / SPAN) * CK * SPAN + (kk * 32) % SPAN;
              const uint32_t off_q = ((kk * 32) / SPAN) * NQ * SPAN + (kk * 32) % SPAN;
              umma_f8_ss(tmem + S::TM_S + (gj & 1) * NQ, dk + (off_k >> 4), dq + (off_q >> 4), IDESC_QK,
                         kk > 0 ? 1u : 0u);
            }
            umma_commit(SFULL(gj & 1));
            umma_commit(KEMPTY(s));
            if (j == n - 1) umma_commit(QEMPTY(qb));
          }
          __syncwarp();
        }
        if (j > 0) {  // O of chunk j - 1
          const int gj = g + j - 1, s = gj % NV;
          ok = paged_wait(PFULL(gj % NPB), (gj / NPB) & 1, failed, 813);
          if (ok) ok = paged_wait(VFULL(s), (gj / NV) & 1, failed, 814);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          if (leader) {
            const uint64_t dp = smem_desc(sbase + S::OFF_P + (gj % NPB) * S::P_BYTES, 16, 8 * S::PM, swizzle_code(S::PM));
            const uint64_t dv = smem_desc(sbase + S::OFF_V + s * S::TILE, CK * SPAN, 8 * SPAN, SWZ);
#pragma unroll
            for (int kk = 0; kk < CK / 32; ++kk)
              umma_f8_ss(tmem + S::TM_O, dp + static_cast<uint64_t>((kk * 32 * S::PM) >> 4),
                         dv + static_cast<uint64_t>((kk * 32 * SPAN) >> 4), IDESC_PV,
                         (j > 1 || kk > 0) ? 1u : 0u);
            umma_commit(PDONE(gj % NPB));
            umma_commit(VEMPTY(s));
          }
          __syncwarp();
        }
      }
      g += n;
    }
    if (leader) {
      umma_commit(BAR_DRAIN);
      paged_wait_drain(BAR_DRAIN, 0, 815);
    }
    __syncwarp();
  } else if (warp == 6) {
    // ------------------------------------------------------------------ fragments and queries
    const int D = p.D, half = D >> 1;
    // A unit's query rows and its rows of the tables come to shared memory, a fragment ahead; then a
    // lane takes element pairs 2 l + 64 e of each half of a head, SETS heads (by lanes, and the
    // same work of several side by side, its loads before all stores: a head's chain alone is some
    // 600 clocks) in each turn of a loop whose code is fetched once.
    constexpr int EPL = DP >= 128 ? DP / 128 : 1;
    constexpr int LPH = DP >= 128 ? 32 : DP / 4;  // lanes per head
    constexpr int HPL = 32 / LPH;                 // heads by lanes
    constexpr int SETS = HPU <= HPL ? 1 : (HPU / HPL < 4 / EPL ? HPU / HPL : 4 / EPL);
    const int ql = lane % LPH, qh = lane / LPH;
    auto widen = [&](uint32_t w) -> float2 { return p.bf16 ? unpack2<true>(w) : unpack2<false>(w); };
    // Rows of the query tiles beyond the parts stay zero.
    for (int i = lane; i < 2 * S::Q_BYTES / 16; i += 32)
      st_shared_v4(sbase + S::OFF_Q + 16 * i, make_uint4(0, 0, 0, 0));
    __syncwarp();
    // Entry k is published before the queries of entry k - 1 are prepared.
    bool ended = false;
    for (int k = 0;; ++k) {
      if (!ended) {
        PagedFrag f;
        ended = !walk.next(p, f);
        if (ended) f.kind = 0;
        const int e = k % S::NF;
        // The producers will ask for these entries of the block table.
        if (!ended && f.kbeg + (lane << p.block_log2) < f.kbeg + f.keys)
          prefetch_l1(p.table + static_cast<long long>(f.b) * p.width + (f.kbeg >> p.block_log2) + lane);
        if (k >= S::NF && !__all_sync(0xffffffffu, paged_wait(FEMPTY(e), ((k / S::NF) - 1) & 1, failed, 821))) break;
        if (lane == 0) {
          *reinterpret_cast<PagedFrag*>(sgen + S::OFF_FRAG + e * 64) = f;
          mbar_arrive(FFULL(e));
        }
        __syncwarp();  // (and every lane is done with the raw rows of entry k - 2)
        if (!ended) {
          if (f.chunks > 0) {
            const uint32_t raw = sbase + S::OFF_RAW + (k & 1) * S::RAW_BYTES;
            const uint8_t* qrow = static_cast<const uint8_t*>(p.q) + (static_cast<long long>(f.b) * p.Hq + f.h0) * (2 * D);
            const long long trow = static_cast<long long>(f.len - 1) * D;
            for (int i = lane; i < f.nh * (D >> 3); i += 32) cp_async16(raw + 16 * i, qrow + 16 * i);
            if (lane < 2 * (D >> 4)) {  // cos, then sin: D bytes each
              const int half16 = D >> 4;
              const bool is_sin = lane >= half16;
              cp_async16(raw + HPU * 2 * D + 16 * lane,
                         static_cast<const uint8_t*>(is_sin ? p.sin : p.cos) + trow + 16 * (is_sin ? lane - half16 : lane));
            }
          }
          cp_async_commit();
        }
      }
      if (k == 0) continue;
      const int it = k - 1, qb = it & 1;
      // (entry k - 1 stays until the softmax warps have read it, which wait for its queries)
      const PagedFrag f = *reinterpret_cast<const PagedFrag*>(sgen + S::OFF_FRAG + (it % S::NF) * 64);
      if (f.kind == 0) break;
      const bool busy = f.chunks > 0;
      // (all but the newest group of copies: entry k - 1's)
      if (ended) cp_async_wait_all(); else cp_async_wait_but_one();
      __syncwarp();
      const uint32_t* raw32 = reinterpret_cast<const uint32_t*>(sgen + S::OFF_RAW + (it & 1) * S::RAW_BYTES);
      if (it >= 2 && !__all_sync(0xffffffffu, paged_wait(QEMPTY(qb), ((it >> 1) - 1) & 1, failed, 820))) break;
      if (busy) {
        uint8_t* qt = sgen + S::OFF_Q + qb * S::Q_BYTES;
        float2 cc[EPL], ss[EPL];
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const int d = 2 * ql + 64 * e;
          cc[e] = widen(d < half ? raw32[(HPU * D + d) >> 1] : 0u);
          ss[e] = widen(d < half ? raw32[(HPU * D + half + d) >> 1] : 0u);
        }
#pragma unroll 1
        for (int h0 = 0; h0 < HPU; h0 += SETS * HPL) {
          float2 y1[SETS][EPL], y2[SETS][EPL];
          uint32_t bits[SETS];
#pragma unroll
          for (int i = 0; i < SETS; ++i) {
            const int h = h0 + i * HPL + qh;
            float top = 0.f;
            bool fine = true;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
              const int d = 2 * ql + 64 * e;
              const bool on = d < half && h < f.nh;
              const float2 a = widen(on ? raw32[(h * D + d) >> 1] : 0u), b = widen(on ? raw32[(h * D + half + d) >> 1] : 0u);
              y1[i][e] = make_float2(a.x * cc[e].x - b.x * ss[e].x, a.y * cc[e].y - b.y * ss[e].y);
              y2[i][e] = make_float2(b.x * cc[e].x + a.x * ss[e].x, b.y * cc[e].y + a.y * ss[e].y);
              top = max3(top, fabsf(y1[i][e].x), fabsf(y1[i][e].y));
              top = max3(top, fabsf(y2[i][e].x), fabsf(y2[i][e].y));
              fine = fine && y1[i][e].x - y1[i][e].x == 0.f && y1[i][e].y - y1[i][e].y == 0.f &&
                     y2[i][e].x - y2[i][e].x == 0.f && y2[i][e].y - y2[i][e].y == 0.f;
            }
            bits[i] = fine ? __float_as_uint(top) : 0x7fc00000u;
          }
          if constexpr (LPH == 32) {
#pragma unroll
            for (int i = 0; i < SETS; ++i) bits[i] = __reduce_max_sync(0xffffffffu, bits[i]);
          } else {
#pragma unroll
            for (int o = LPH / 2; o >= 1; o >>= 1)
#pragma unroll
              for (int i = 0; i < SETS; ++i) bits[i] = max(bits[i], __shfl_xor_sync(0xffffffffu, bits[i], o));
          }
#pragma unroll
          for (int i = 0; i < SETS; ++i) {
            // a power of two: the row divided by it fits e4m3 (NaN for a row that is not finite, whose
            // scores the factor makes NaN)
            const float u = paged_unit(bits[i]);
            const float inv = __uint_as_float(0x7f000000u - __float_as_uint(u));  // 1 / u
            const int h = h0 + i * HPL + qh;
            if (ql == 0 && h < HPU) reinterpret_cast<float*>(sgen + S::OFF_QS)[qb * HPU + h] = u * p.scale_log2;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
              y1[i][e] = make_float2(y1[i][e].x * inv, y1[i][e].y * inv);
              y2[i][e] = make_float2(y2[i][e].x * inv, y2[i][e].y * inv);
            }
          }
#pragma unroll
          for (int t = 0; t < 3; ++t) {
#pragma unroll
            for (int i = 0; i < SETS; ++i) {
              const int h = h0 + i * HPL + qh;
#pragma unroll
              for (int e = 0; e < EPL; ++e) {
                const int d = 2 * ql + 64 * e;
                float2 &v1 = y1[i][e], &v2 = y2[i][e];
                const uint32_t p1 = e4m3x2(v1.x, v1.y), p2 = e4m3x2(v2.x, v2.y);
                if (t < 2) {
                  const float2 w1 = e4m3x2_widen(p1), w2 = e4m3x2_widen(p2);
                  v1 = make_float2((v1.x - w1.x) * 16.0f, (v1.y - w1.y) * 16.0f);
                  v2 = make_float2((v2.x - w2.x) * 16.0f, (v2.y - w2.y) * 16.0f);
                }
                if (d < half && h < HPU) {
                  // row t HPU + h of the tile: swizzled, K-major
                  const int n = t * HPU + h, d2 = d + half;
                  *reinterpret_cast<uint16_t*>(qt + swz_chunk_offset<SPAN>(NQ, n, d >> 4) + (d & 15)) =
                      static_cast<uint16_t>(p1);
                  *reinterpret_cast<uint16_t*>(qt + swz_chunk_offset<SPAN>(NQ, n, d2 >> 4) + (d2 & 15)) =
                      static_cast<uint16_t>(p2);
                }
              }
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();  // (and the raw rows have been read)
      if (lane == 0) mbar_arrive(QFULL(qb));
    }
    // Lengths out of range are reported by the first CTA, once its work is under way.
    if (blockIdx.x == 0)
      for (int b = lane; b < p.B; b += 32)
        if (static_cast<unsigned>(p.lens[b]) > static_cast<unsigned>(p.max_len))
          record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(p.lens[b]));
  } else {
    // ------------------------------------------------------------------ warps 0-3: softmax
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    bool ok = true;
    int g = 0, mq = 0, nf = 0;  // chunks, combined column blocks, fragments with keys
    for (int it = 0; ok; ++it) {
      const int qb = it & 1;
      if (!(ok = __all_sync(0xffffffffu, softmax_wait<DP>(FFULL(it % S::NF), (it / S::NF) & 1, failed, 829)))) break;
      const PagedFrag f = *reinterpret_cast<const PagedFrag*>(sgen + S::OFF_FRAG + (it % S::NF) * 64);
      if (f.kind == 0) break;
      if (!(ok = __all_sync(0xffffffffu, softmax_wait<DP>(QFULL(qb), (it >> 1) & 1, failed, 830)))) break;
      float qs[HPU];
#pragma unroll
      for (int h = 0; h < HPU; ++h) qs[h] = reinterpret_cast<const float*>(sgen + S::OFF_QS)[qb * HPU + h];
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(QEMPTY(qb));
        mbar_arrive(FEMPTY(it % S::NF));
      }
      auto store_out = [&](long long row, int d, float val) {
        if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[row * p.D + d] = __float2bfloat16_rn(val);
        else static_cast<__half*>(p.out)[row * p.D + d] = __float2half_rn(val);
      };
      const long long row0 = static_cast<long long>(f.b) * p.Hq + f.h0;
      if (f.chunks == 0) {
        for (int i = tid; i < f.nh * p.D; i += 128) store_out(row0 + i / p.D, i % p.D, 0.f);
        if (tid == 0) *emitted = it + 1;
        continue;
      }
      // A key's row of P has only its warp's bytes (a 16- or 32-byte part); the rest is zero, once
      // the last fragment's rows of O, which lie there too, have been read.
      if (mq > 0 && !(ok = __all_sync(0xffffffffu, softmax_wait<DP>(BAR_FREE, (mq - 1) & 1, failed, 838)))) break;
#pragma unroll
      for (int i = 0; i < NPB * S::PM / 16; ++i)
        st_shared_v4(sbase + S::OFF_P + (i / (S::PM / 16)) * S::P_BYTES + warp * 32 * S::PM + 512 * (i % (S::PM / 16)) + 16 * lane,
                     make_uint4(0, 0, 0, 0));
      __syncwarp();  // (a warp's rows lie together, and only its own threads write them)
      float m[HPU], l[HPU];
#pragma unroll
      for (int h = 0; h < HPU; ++h) {
        m[h] = -FLT_MAX;  // (not infinite: a masked key's weight is 2^(-inf - m) = 0)
        l[h] = 0.f;
      }
      for (int j = 0; j < f.chunks; ++j) {
        const int gj = g + j, s = gj % NK;
        const int left = f.keys - j * CK;  // keys of this chunk and those behind it
        const bool valid = tid < left;
        ok = softmax_wait<DP>(KFULL(s), (gj / NK) & 1, failed, 831);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        const float* sc = reinterpret_cast<const float*>(sgen + S::OFF_SC + s * 64);
        const float ksc = valid ? sc[tid >> p.block_log2] : 1.0f;
        float vsc = valid ? sc[8 + (tid >> p.block_log2)] : 1.0f;
        if (vsc < 0x1p-64f) vsc = 0x1p-64f;  // (the writer's smallest; a NaN stays)
        __syncwarp();
        if (lane == 0) mbar_arrive(KEMPTY(s));
        const float lv = lg2(vsc), lsum = lv - 24.0f;
        ok = softmax_wait<DP>(SFULL(gj & 1), (gj >> 1) & 1, failed, 832);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        float sv[NQ];
#pragma unroll
        for (int c = 0; c < NQ; c += 16) tmem_ld16(tmem + lane_off + S::TM_S + (gj & 1) * NQ + c, sv + c);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(SEMPTY(gj & 1));
        float u[HPU];
        bool over = false;
#pragma unroll
        for (int h = 0; h < HPU; ++h) {
          const float dot = fmaf(sv[2 * HPU + h], 0x1p-8f, fmaf(sv[HPU + h], 0x1p-4f, sv[h]));
          u[h] = valid ? fmaf(dot, qs[h] * ksc, lv) : -INFINITY;
          over |= u[h] > m[h] + 8.0f;
        }
        float alpha[HPU];
        const bool moved = __any_sync(0xffffffffu, over);
        if (moved) {
#pragma unroll
          for (int h = 0; h < HPU; ++h) {
            const float mx = warp_max(u[h]);
            const float mn = mx > m[h] + 8.0f ? mx - DECODE_PAGED_BELOW : m[h];
            // (in two halves: where the value scales jump the factor alone may be less than any float)
            const float a = ex2(0.5f * (m[h] - mn));
            alpha[h] = a * a;
            l[h] = l[h] * a * a;
            m[h] = mn;
          }
        }
        float pe[HPU];
#pragma unroll
        for (int h = 0; h < HPU; ++h) {
          const float x = u[h] - m[h];
          pe[h] = ex2(x);
          l[h] += ex2(x - lsum);
        }
        // Parts of the weights, rows t HPU + h of this warp: 4 HPU bytes of the key's row of P.
        uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if constexpr (HPU == 1) {
          uint32_t t[4];
          e4m3_parts2(pack2<false>(pe[0], 0.f), t);
          w[0] = (t[0] & 0xffu) | ((t[1] & 0xffu) << 8) | ((t[2] & 0xffu) << 16) | (t[3] << 24);
        } else if constexpr (HPU == 2) {
          uint32_t t[4];
          e4m3_parts2(pack2<false>(pe[0], pe[1]), t);
          w[0] = t[0] | (t[1] << 16);
          w[1] = t[2] | (t[3] << 16);
        } else {
#pragma unroll
          for (int h = 0; h < HPU; h += 4) {
            uint32_t a[4], b[4];
            e4m3_parts2(pack2<false>(pe[h], pe[h + 1]), a);
            e4m3_parts2(pack2<false>(pe[h + 2], pe[h + 3]), b);
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t * (HPU / 4) + h / 4] = a[t] | (b[t] << 16);
          }
        }
        // The P buffer was last read by PV(gj - NPB); a moved reference rescales O, which holds PV up
        // to gj - 1 of this fragment.
        if (gj >= NPB) ok = softmax_wait<DP>(PDONE(gj % NPB), ((gj / NPB) - 1) & 1, failed, 833);
        if (NPB > 1 && ok && moved && j > 0) ok = softmax_wait<DP>(PDONE((gj - 1) % NPB), ((gj - 1) / NPB) & 1, failed, 834);
        if (ok && left < CK) ok = softmax_wait<DP>(VFULL(gj % NV), (gj / NV) & 1, failed, 835);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        if (moved && j > 0) {
          float al = 1.0f;
#pragma unroll
          for (int h = 0; h < HPU; ++h) al = (lane % HPU) == h ? alpha[h] : al;
          // (a row that was zero and whose reference was none yet: alpha is 0, O is 0)
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            float o[16];
            tmem_ld16(tmem + lane_off + S::TM_O + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= al;
            tmem_st16(tmem + lane_off + S::TM_O + c, o);
          }
          tmem_wait_st();
        }
        const uint32_t pbuf = sbase + S::OFF_P + (gj % NPB) * S::P_BYTES;
        st_shared_v4(pbuf + swz_chunk_offset<S::PM>(CK, tid, warp * (S::PM / 64)), make_uint4(w[0], w[1], w[2], w[3]));
        if constexpr (S::PM == 128)
          st_shared_v4(pbuf + swz_chunk_offset<S::PM>(CK, tid, 2 * warp + 1), make_uint4(w[4], w[5], w[6], w[7]));
        if (!valid) {
          // Rows behind the last key may hold anything, a NaN among it, and 0 x NaN is a NaN.
          // (the lanes begin at different 16 bytes of their rows: no two in the same banks)
          constexpr int PER = SPAN / 16;
          const int turn = tid / (8 / PER) % PER;
#pragma unroll
          for (int c = 0; c < DP / 16; ++c)
            st_shared_v4(sbase + S::OFF_V + (gj % NV) * S::TILE + (c / PER) * CK * SPAN + tid * SPAN + 16 * (c % PER ^ turn),
                         make_uint4(0, 0, 0, 0));
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();  // (one arrival per warp: 32 on one barrier take their turns)
        if (lane == 0) mbar_arrive(PFULL(gj % NPB));
      }
      if (!ok) break;
      g += f.chunks;
      // Sums of the weights: the lanes' sums of HPU heads, halving the heads with the lanes.
      {
        int n = HPU;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          if (n > 1) {
            n >>= 1;
#pragma unroll
            for (int h = 0; h < HPU / 2; ++h)
              if (h < n) {
                const float send = (lane & o) ? l[h] : l[h + n], keep = (lane & o) ? l[h + n] : l[h];
                l[h] = keep + __shfl_xor_sync(0xffffffffu, send, o);
              }
          } else {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
          }
        }
      }
      // Maxima and sums of the warps, exchanged while the last PV runs.
      {
        // The head of a lane's sum: its top log2(HPU) lane bits.
        constexpr int LANES = 32 / HPU;
        if (lane % LANES == 0) mrg_l[warp * HPU + lane / LANES] = l[0];
        float mm = m[0];
#pragma unroll
        for (int h = 1; h < HPU; ++h) mm = lane == h ? m[h] : mm;
        if (lane < HPU) mrg_m[warp * HPU + lane] = mm;
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR_ML);
      }
      float* part_o = p.part + static_cast<long long>(f.slot) * HPU * p.D;
      if (!(ok = __all_sync(0xffffffffu, softmax_wait<DP>(BAR_ML, nf++ & 1, failed, 837)))) break;
      // Lane t HPU + h: the factor of this warp's row of it, 2^(m_w - M) / L 2^(-5 t).
      float wt;
      {
        const int i = lane % (4 * HPU);  // warp w HPU + head
        const float mi = mrg_m[i];
        float top = fmaxf(mi, __shfl_xor_sync(0xffffffffu, mi, HPU));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2 * HPU));
        const float half_fac = ex2(0.5f * (mi - top));  // (as above)
        float fac = half_fac * half_fac;
        float L = mrg_l[i] * half_fac * half_fac;
        L += __shfl_xor_sync(0xffffffffu, L, HPU);
        L += __shfl_xor_sync(0xffffffffu, L, 2 * HPU);
        fac = fac * 0x1p24f / L;
        if (f.nf > 1 && tid < HPU) p.part[(2LL * gridDim.x * p.D + f.slot) * HPU + tid] = top + (lg2(L) - 24.0f);  // log2 of the sum
        const int t = lane / HPU & 3;
        wt = __shfl_sync(0xffffffffu, fac, warp * HPU + lane % HPU) * __int_as_float((127 - 5 * t) << 23);
      }
      // Combine the warps' rows of O, CB columns at a time: rows 32 w + t HPU + h under their factors
      // through shared memory, then a thread sums the 16 of an output.
      if (!(ok = __all_sync(0xffffffffu, softmax_wait<DP>(PDONE((g - 1) % NPB), ((g - 1) / NPB) & 1, failed, 836)))) break;
      tc_fence_after();
#pragma unroll 1
      for (int cb = 0; cb < DP && ok; cb += S::CB) {
        {
          float o[S::CB];
#pragma unroll
          for (int c = 0; c < S::CB; c += 16) tmem_ld16(tmem + lane_off + S::TM_O + cb + c, o + c);
          // The columns combined before have been read.
          if (cb > 0) ok = softmax_wait<DP>(BAR_FREE, (mq - 1) & 1, failed, 837);
          tmem_wait_ld();
          if (lane < 4 * HPU) {
            // (part i of row r is at i ^ (r & 7): no two of eight rows in the same banks)
            float4* dst = reinterpret_cast<float4*>(mrg + (warp * 4 * HPU + lane) * CB);
            const int turn = (warp * 4 * HPU + lane) & 7;
#pragma unroll
            for (int i = 0; i < CB / 4; ++i)
              dst[i ^ turn] = make_float4(o[4 * i] * wt, o[4 * i + 1] * wt, o[4 * i + 2] * wt, o[4 * i + 3] * wt);
          }
        }
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR_MRG);
        if (!(ok = __all_sync(0xffffffffu, softmax_wait<DP>(BAR_MRG, mq & 1, failed, 837)))) break;
        // A thread takes a column and every (128 / columns)-th head.
        const int nd_log2 = p.D >= S::CB ? (S::CB == 64 ? 6 : 5) : 4;  // (4: head_dim 16)
        const int d = tid & ((1 << nd_log2) - 1), hg = tid >> nd_log2;
        const int hs = 128 >> nd_log2;
        constexpr int NH = HPU * S::CB > 128 ? HPU * S::CB / 128 : 1;  // a thread's heads (less at head_dim 16)
        float A[NH];
#pragma unroll
        for (int i = 0; i < NH; ++i) {
          const int h = (hg + i * hs) & (HPU - 1);  // (taken round where there are fewer)
          A[i] = 0.f;
#pragma unroll
          for (int w2 = 0; w2 < 4; ++w2) {
            float part[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int row = (w2 * 4 + t) * HPU + h;
              part[t] = mrg[row * CB + 4 * ((d >> 2) ^ (row & 7)) + (d & 3)];
            }
            A[i] += ((part[3] + part[2]) + part[1]) + part[0];
          }
        }
#pragma unroll
        for (int i = 0; i < NH; ++i) {
          const int h = hg + i * hs;
          if (h < f.nh) {
            if (f.nf == 1) store_out(row0 + h, cb + d, A[i]);
            else part_o[h * p.D + cb + d] = A[i];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR_FREE);
        ++mq;
      }
      if (!ok) break;
      if (tid == 0) {
        if (f.nf > 1) {
          // A ticket on the unit's counter. The partial stores reach this thread through the barrier;
          // its acquire-release add makes them visible before the ticket and, after the last
          // ticket, the other fragments' partials visible to this CTA.
          if (softmax_wait<DP>(BAR_FREE, (mq - 1) & 1, failed, 839)) {
            if (atom_add_acq_rel_gpu(&p.cnt[f.c0], 1) == f.nf - 1) {
              p.cnt[f.c0] = 0;  // no other ticket is to come: ready for the next call
              owed[*n_owed] = f;
              *n_owed = *n_owed + 1;
            }
            *emitted = it + 1;
          }
        } else {
          *emitted = it + 1;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // Units whose last ticket was this CTA's, of its first and its last fragment at most. A thread takes
  // four columns of a head at a time; the rows of the first KB fragments are on their way while
  // the weights are found, a warp per head, a lane per fragment.
  for (int e = 0; e < *n_owed; ++e) {
    const PagedFrag f = owed[e];
    constexpr int KB = 8;
    auto slot_of = [&](int k) { return k == 0 ? 2 * f.c0 + 1 : 2 * (f.c0 + k); };
    // `groups` threads of a warp share an output's fragments: k = group, group + groups, ...
    const int q4 = p.D >> 2, items = f.nh * q4;
    int groups_log2 = 0;
    while ((items << (groups_log2 + 1)) <= S::NTHREADS && (2 << groups_log2) <= f.nf && groups_log2 < 5) ++groups_log2;
    const int groups = 1 << groups_log2;
    auto load = [&](float4 (&o)[KB], int i, int k0) {
      const int h = small_div(i, q4), d = 4 * (i - h * q4);
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int kk = k0 + (k << groups_log2);
        if (i < items && kk < f.nf)
          o[k] = __ldcg(reinterpret_cast<const float4*>(
              p.part + (static_cast<long long>(slot_of(kk)) * HPU + h) * p.D + d));
      }
    };
    const int group = tid & (groups - 1);
    float4 o[KB];
    load(o, tid >> groups_log2, group);
    const float* part_l = p.part + 2LL * gridDim.x * HPU * p.D;
    float* wt = mrg;  // [HPU][nf]: nf <= gridDim.x <= DECODE_PAGED_MAX_CTAS
    for (int h = warp; h < f.nh; h += S::NTHREADS / 32) {
      float M = -INFINITY, L = 0.f;
      for (int k = lane; k < f.nf; k += 32) {
        const float x = __ldcg(part_l + slot_of(k) * HPU + h);
        wt[h * f.nf + k] = x;
        M = fmaxf(M, x);
      }
      M = warp_max(M);
      for (int k = lane; k < f.nf; k += 32) {
        const float x = ex2(wt[h * f.nf + k] - M);
        wt[h * f.nf + k] = x;
        L += x;
      }
#pragma unroll
      for (int o2 = 16; o2 >= 1; o2 >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o2);
      const float inv = 1.0f / L;
      for (int k = lane; k < f.nf; k += 32) wt[h * f.nf + k] *= inv;
    }
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += S::NTHREADS >> groups_log2) {
      const int i = i0 + (tid >> groups_log2);
      const int h = small_div(i, q4), d = 4 * (i - h * q4);
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < items) {
#pragma unroll 1
        for (int k0 = group; k0 < f.nf; k0 += KB << groups_log2) {
          if (i0 > 0 || k0 > group) load(o, i, k0);
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            const int kk = k0 + (k << groups_log2);
            if (kk >= f.nf) break;
            const float x = wt[h * f.nf + kk];
            A.x = fmaf(o[k].x, x, A.x);
            A.y = fmaf(o[k].y, x, A.y);
            A.z = fmaf(o[k].z, x, A.z);
            A.w = fmaf(o[k].w, x, A.w);
          }
        }
      }
      for (int o2 = 1; o2 < groups; o2 <<= 1) {  // (an output's threads are neighbours in a warp)
        A.x += __shfl_xor_sync(0xffffffffu, A.x, o2);
        A.y += __shfl_xor_sync(0xffffffffu, A.y, o2);
        A.z += __shfl_xor_sync(0xffffffffu, A.z, o2);
        A.w += __shfl_xor_sync(0xffffffffu, A.w, o2);
      }
      if (i >= items || group != 0) continue;
      const long long at = (static_cast<long long>(f.b) * p.Hq + f.h0 + h) * p.D + d;
      uint2 w;
      if (p.bf16) w = make_uint2(pack2<true>(A.x, A.y), pack2<true>(A.z, A.w));
      else w = make_uint2(pack2<false>(A.x, A.y), pack2<false>(A.z, A.w));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = w;
    }
    __syncthreads();
  }
  if (*failed) {
    // A wait ran out (reported in the status words): NaN for what this CTA still owes, and its
    // tickets, so that the counters return to zero.
    walk.init(*start);
    PagedFrag f;
    const float nan = __int_as_float(0x7fc00000);
    for (int it = 0; walk.next(p, f); ++it) {
      if (it < *emitted) continue;
      for (int i = tid; i < f.nh * p.D; i += S::NTHREADS) {
        const int h = i / p.D, d = i - h * p.D;
        const long long o = (static_cast<long long>(f.b) * p.Hq + f.h0 + h) * p.D + d;
        if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(nan);
        else static_cast<__half*>(p.out)[o] = __float2half_rn(nan);
        if (f.nf > 1) {
          p.part[(static_cast<long long>(f.slot) * HPU + h) * p.D + d] = nan;
          if (d == 0) p.part[2LL * gridDim.x * HPU * p.D + f.slot * HPU + h] = nan;
        }
      }
      __threadfence();
      __syncthreads();
      if (f.nf > 1 && tid == 0 && atom_add_acq_rel_gpu(&p.cnt[f.c0], 1) == f.nf - 1) p.cnt[f.c0] = 0;
    }
  }
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

}  // namespace du
