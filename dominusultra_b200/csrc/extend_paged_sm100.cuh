// Attention of several new tokens per request over the paged 8-bit KV cache (layout in
// paged_sm100.cuh), on tcgen05.
//
// Request b has past_b tokens cached before its n_b = len_b - past_b new ones, which are cached too. For
// its new token t and query head h of KV head g:
//   q' = R(past_b + t) q    s_j = (q' . k8_j) ks[page_j, g] scale    j <= past_b + t
//   out = sum_j softmax(s)_j v8_j vs[page_j, g]
// Rows t >= n_b are zeros.
//
// Rows: the G query heads of a KV head share its keys, so the rows of (b, g) are numbered t G + h and
// cut into items of up to 256 rows, whatever tokens and heads those are. Keys go in tiles of KT. Both
// products are kind::f16: the cached bytes are widened to fp16 (exactly, by one conversion per pair) in
// shared memory once per tile for all rows of an item, unscaled. Scales are per block of at least 16
// keys, so they cost a multiplication per 16 scores: with x = s + log2 vs (log2 domain, s = S kq, kq the
// key scale, the softmax scale and the query row's own factor) the carried weight is 2^(x - m + 8) =
// w vs up to a row's constant, an fp16 value of at most 2^15 since m moves when some x exceeds it by 7,
// and the sum takes 2^(vr - log2 vs) times the sum of a group's weights, vr being the log2 of the first
// value scale of the fragment. Where a value scale is beyond 2^30 of that (then, and for the rest of the
// fragment) the sum has exponentials and a reference of its own: a key whose carried weight is nothing
// beside another's can have all of the softmax's. fp16 holds weights down to 2^-22 of a row's largest at
// full precision, and half its smallest step is 2^-33 of that. Query rows are carried as fp16 with a power of two for each row.
//
// Work: the items' key tiles, item by item, cut into equal ranges, one per CTA of a persistent grid (an
// item's beginning is charged with PEN tiles). Lengths are read on the device; every CTA repeats the sum
// over them. An item within one CTA is written at once; the fragments of others leave fp32 partials, which
// a second kernel joins with all SMs (a CTA that joined its item's five fragments of 256 rows took 20-30 us
// for it at the end of a call, when the others were done).
//
// Streams: two softmax warpgroups (one at head_dim 256, where tensor memory holds one O), each with an O and a
// warp that issues its products. P overwrites its S.
//  - NT = 2 (more than 128 rows in an item): a stream is a tile of 128 rows. It has two tiles of S of 64 keys, so
//    that a warpgroup goes from tile to tile without waiting for products (also at head_dim 256, with one row tile).
//  - NT = 1: the streams share the one row tile and take every other key tile of 128 each; a row then has two
//    parts, each with a maximum, sum and O of its own, joined at the fragment's end. Of the bytes that widening and
//    products move through shared memory the query rows' are per tile, and so are the hand-offs, so tiles are long
//    (with 64 keys 117 -> 122 us for 16 requests of 128 rows behind 10000 keys), and the other stream's softmax
//    fills the time in which one waits.
//  - Copies: a softmax warp has 32 of the row tile's rows, so with 64 rows or fewer most would idle while one has all
//    the keys of a tile to do: there the tile holds two (or, with 32 rows, four) copies of the rows, and a copy's
//    warps take half (a quarter) of each tile's keys, P being zero for the others. Each copy is a part of its
//    rows of its own. (At head_dim 256 joining the copies cost as much as they gave.)
//
// Bounds and measures (device time): where a stream has its own rows, the exponentials and what a warp does
// around them: of the ~2400 clocks that a stream takes for 128 rows and 64 keys 512 are the special function
// unit's, ~600 other instructions of the same warp and the rest waits (32 heads on 8 of 128: the last 2048 of
// 32768 tokens 1.20 ms, 890 TFLOP/s, 54 % of a bf16 product's rate; 256 behind 32512 177 us; 8 requests of up to
// 777 tokens, 32 heads of 64, up to 2048 keys 165 us). Where streams share rows, latency too (no unit is half
// busy), then shared memory: per 128 keys at head_dim 128 it moves 32 KB raw in and out, 64 KB widened in and out
// again and the query rows' 32 KB, at least ~1800 clocks against 1400 that the cached bytes take from HBM; then the
// beginnings and ends of fragments, ~10000 clocks each (64 requests of up to 4096, 4 new tokens, 32 heads on 8 of
// 128: 109 us, 2.5 TB/s; 16 of up to 20001, 16 tokens, 64 on 8: 115 us). These are the bounds of this schedule: the
// single-token kernel, which feeds cached bytes to the tensor cores as they are, streams such caches in half the
// time. A small call is its launches and a chain of dependent loads (8.5 us where one key tile covers the table's
// row, so that nothing is to be joined).
//
// Warps (512 threads): 0-3 and 4-7 softmax; 8-11 widen K and V (4-11 at head_dim 256); 12 bulk copies of K;
// 13 walks the fragments, fetches the scales and copies V; 14 and 15 the products of a stream each (14: and
// TMEM). Every wait is bounded.
#pragma once

#include <float.h>

#include <type_traits>

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
  // Partial outs [2 gridDim.x][D / 4][rows] by four columns (neighbouring lanes have neighbouring rows), then
  // the log2 of their sums, in two parts, [2 gridDim.x][rows].
  float* part;
  int* split;         // [gridDim.x][8]: the item that this CTA has the first of several fragments of
  int max_len;        // tokens that the table's row and the rope tables cover
  int bf16;
  int B, Hq, Hkv, G, T, N, width;
  int items;          // of a request with T new tokens
  int block, block_log2;
  float scale_log2;
};

constexpr int EXTEND_THREADS = 512;
constexpr float EXTEND_TOP = 8.0f;   // log2 of the weight at a row's reference
constexpr float EXTEND_MOVE = 7.0f;   // how far beyond its reference a row's maximum may be
constexpr float EXTEND_LARGE = 1024.0f;  // references beyond this are kept in two parts
constexpr float EXTEND_FAR = 30.0f;   // how far a value scale may be from the fragment's first

template <int D_, int NT_, int CP_ = 1>
struct ExtendShape {
  static constexpr int D = D_, NT = NT_;
  static constexpr int CP = CP_;                 // copies of the row tile's rows
  static constexpr int NS = D <= 128 ? 2 : 1;    // streams
  static constexpr bool ALT = NT < NS;           // that take key tiles in turn
  static constexpr int RP = NT * 128;            // rows of an item
  static constexpr int SB = NT == 2 || D == 256 ? 2 : 1;  // tiles of S of a stream
  static constexpr int KT = SB == 2 ? 64 : 128;  // keys of a tile
  static constexpr int SPAN = 2 * D >= 128 ? 128 : 2 * D;  // bytes per row of a swizzled block
  static constexpr int GPT = KT / 16;            // groups of 16 keys in a tile
  static constexpr int NB = 32 / GPT;            // tiles of a batch of scales
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int T_BYTES = KT * D * 2;     // a widened tile
  static constexpr int RK = 64;                  // keys of a copied piece
  static constexpr int RPT = KT / RK;            // pieces of a tile
  static constexpr int RAW = RK * D;
  static constexpr int NK = D == 256 || SB == 1 ? 2 : 3, NV = D == 256 ? 1 : NK;  // widened tiles
  static constexpr int MISC = 2048;
  static constexpr int RAWS = (231424 - MISC - NT * Q_BYTES - (NK + NV) * T_BYTES) / RAW;
  static constexpr int NRV = RAWS / 2 > 8 ? 8 : RAWS / 2;             // copied pieces of V in flight
  static constexpr int NRK = RAWS - NRV > 8 ? 8 : RAWS - NRV;         // and of K
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + NT * Q_BYTES;
  static constexpr int OFF_V = OFF_K + NK * T_BYTES;
  static constexpr int OFF_RK = OFF_V + NV * T_BYTES;
  static constexpr int OFF_RV = OFF_RK + NRK * RAW;
  static constexpr int OFF_MISC = OFF_RV + NRV * RAW;
  static constexpr int NF = 3;                         // fragment entries in flight
  static constexpr int OFF_SC = OFF_MISC;              // [2] batches of scales
  static constexpr int SC_BYTES = 3 * 128 + 4 * NB + 16;  // kq, log2 vs, factor [32]; zero mask [NB]; vr, far
  static constexpr int OFF_FRAG = OFF_SC + 2 * SC_BYTES;
  static constexpr int OFF_BAR = OFF_FRAG + NF * 64;
  static constexpr int B_RKF = 0, B_RKE = B_RKF + NRK, B_RVF = B_RKE + NRK, B_RVE = B_RVF + NRV, B_KF = B_RVE + NRV,
                       B_KE = B_KF + NK, B_VF = B_KE + NK, B_VE = B_VF + NV, B_SCF = B_VE + NV, B_SCE = B_SCF + 2,
                       B_QF = B_SCE + 2, B_SF = B_QF + 2, B_PF = B_SF + 4, B_OF = B_PF + 4, B_OD = B_OF + 2,
                       B_FF = B_OD + 2, B_FE = B_FF + NF, B_DR = B_FE + NF, N_BAR = B_DR + 2;
  static constexpr int OFF_WORDS = OFF_BAR + 8 * N_BAR;  // TMEM address, failed
  static constexpr int SMEM_BYTES = OFF_WORDS + 16 + 1024;
  static constexpr int TM_S = 0;             // + (SB x + tile % SB) KT, x the stream
  static constexpr int TM_O = NS * SB * KT;  // + x D
  static constexpr int TMEM_COLS = TM_O + NS * D <= 256 ? 256 : 512;
  static constexpr int SW = 4 * NS;      // softmax warps
  static constexpr int WC = NS == 2 ? 2 : 4;  // warps that widen K, and as many V
  static constexpr int REG_SOFTMAX = 200, REG_WIDEN = NS == 2 ? 64 : 112, REG_ISSUE = NS == 2 ? 48 : 88;
  // Tiles that an item's beginning is charged with. (Of 128 keys, with 4 / 5 / 7: 64 requests of up to 4096 111 /
  // 109 / 105 us, 128 of 1000 110 / 116 / 117, 16 of up to 20001 116 / 115 / 117, 16 of 2048 at head_dim 64 84 /
  // 79 / 80; of 64 keys, with 4 / 5 / 6: 163 / 163 / 164, 256 tokens behind 32512 180 / 179 / 178.)
  static constexpr int PEN = KT == 64 ? 6 : 5;
  static constexpr int KC = KT / CP;             // keys of a tile that a softmax warp takes
  static constexpr int RW = 4 / CP;              // softmax warps of a copy
  static constexpr int PARTS = CP * (ALT ? NS : 1);  // of a row, to be joined
  static_assert(NT <= NS, "a row tile needs a stream");
  static_assert(CP == 1 || (NT == 1 && (CP == 2 || CP == 4) && KC % 16 == 0), "copies");
  static_assert(TM_O + NS * D <= 512, "tensor memory");
  static_assert(NRV >= 1 && NRK >= NRV && NB * RPT == 8, "copied pieces in flight");
  static_assert(OFF_WORDS + 16 - OFF_MISC <= MISC && SMEM_BYTES <= 232448, "shared memory budget");
  static_assert(OFF_FRAG % 16 == 0 && OFF_BAR % 8 == 0 && SC_BYTES % 16 == 0 && OFF_MISC % 16 == 0, "alignment");
  static_assert((NS * REG_SOFTMAX + (3 - NS) * REG_WIDEN + REG_ISSUE) * 128 <= EXTEND_THREADS * 128, "register split");
};

// One fragment, as warp 13 leaves it for the other warps (16 words).
struct ExtendFrag {
  int kind;         // 1 a fragment, 0 the end
  int b, kvh;
  int row0, rows;   // the item's first row of (b, kvh), and its rows
  int past, len;
  int j0, j1;       // key tiles
  int nk0, nk1;     // key tiles that the first and the second row tile have (0: no such row tile)
  int nf, c0;       // fragments of the item, CTA of the first
  int slot;         // partial slot when nf > 1
  int pad[2];
};

__device__ __forceinline__ int extend_new(const ExtendPagedParams& p, int b, int& past, int& len) {
  past = p.past[b];
  len = p.lens[b];
  const bool ok = past >= 0 && len >= past && len <= p.max_len && len - past <= p.T;
  return ok ? len - past : (len = past = 0, -1);
}

// Walks a CTA's share of the flattened tiles fragment by fragment (one warp; all lanes hold the same).
// Positions run over requests, items of a request and KV heads, in that order; a KV head's item takes PEN
// positions and one per key tile. The host keeps them below 2^31.
template <typename S>
struct ExtendWalk {
  int cur, hi, base, per, grid;  // base: position of the current item's beginning
  int b, kvh, item, past, len, items, cost;
  // Key tiles of rows up to `row` of (b, kvh).
  __device__ __forceinline__ static int tiles(const ExtendPagedParams& p, int past, int row) { return (past + small_div(row, p.G)) / S::KT + 1; }
  // Positions of an item of request b for one KV head; 0: the request has no such item.
  __device__ __forceinline__ static int span(const ExtendPagedParams& p, int b, int item) {
    int past, len;
    const int rows = max(extend_new(p, b, past, len), 0) * p.G;
    return item * S::RP < rows ? tiles(p, past, min(rows, (item + 1) * S::RP) - 1) + S::PEN : 0;
  }
  // The request's lengths, and the item's cost.
  __device__ __forceinline__ void enter(const ExtendPagedParams& p) {
    const int rows = max(extend_new(p, b, past, len), 0) * p.G;
    items = (rows + S::RP - 1) / S::RP;
  }
  __device__ __forceinline__ void init(const ExtendPagedParams& p, int lane) {
    grid = static_cast<int>(gridDim.x);
    const int most = p.items, pairs = p.B * most;  // items of a request with T new tokens; (request, item)
    auto span_of = [&](int e) {
      if (e >= pairs) return 0;
      const int bb = most == 1 ? e : small_div(e, most);
      return span(p, bb, e - bb * most);
    };
    const int span0 = span_of(lane);  // (most batches have no more)
    int total = span0;
    for (int e = 32 + lane; e < pairs; e += 32) total += span_of(e);
    total = static_cast<int>(__reduce_add_sync(0xffffffffu, total)) * p.Hkv;
    per = max((total + grid - 1) / grid, S::PEN);  // (no cuts so fine that joining costs more)
    cur = static_cast<int>(min(static_cast<long long>(per) * blockIdx.x, static_cast<long long>(total)));
    hi = min(total - cur, per) + cur;
    base = b = kvh = item = items = 0;
    if (cur >= hi) return;
    // The item that holds `cur`.
    for (int e0 = 0; e0 < pairs; e0 += 32) {
      const int own = e0 == 0 ? span0 : span_of(e0 + lane);
      int in = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, cur - base < in * p.Hkv);
      if (hit) {
        const int l = __ffs(static_cast<int>(hit)) - 1;
        cost = __shfl_sync(0xffffffffu, own, l);
        b = most == 1 ? e0 + l : small_div(e0 + l, most);
        item = e0 + l - b * most;
        base += __shfl_sync(0xffffffffu, in - own, l) * p.Hkv;
        kvh = small_div(cur - base, cost);
        base += kvh * cost;
        break;
      }
      base += __shfl_sync(0xffffffffu, in, 31) * p.Hkv;
    }
    enter(p);
  }
  __device__ __forceinline__ bool next(const ExtendPagedParams& p, ExtendFrag& f) {
    while (true) {
      if (cur >= hi) return false;
      const int first = base + S::PEN, end = base + cost;
      const int j0 = max(cur - first, 0), j1 = min(hi, end) - first;
      cur = min(hi, end);
      if (j1 > 0) {
        f.kind = 1;
        f.b = b;
        f.kvh = kvh;
        f.row0 = item * S::RP;
        f.rows = min((len - past) * p.G - f.row0, S::RP);
        f.past = past;
        f.len = len;
        f.j0 = j0;
        f.j1 = j1;
        f.nk0 = tiles(p, past, f.row0 + min(f.rows, 128) - 1);
        f.nk1 = f.rows > 128 ? end - first : 0;
        f.c0 = small_div(first, per);
        f.nf = small_div(end - 1, per) - f.c0 + 1;
        f.slot = 2 * static_cast<int>(blockIdx.x) + (j0 > 0 ? 0 : 1);
      }
      if (cur == end && cur < hi) {
        base = end;
        if (++kvh == p.Hkv) {
          kvh = 0;
          ++item;
          while (item >= items) {  // the next request that has any (there is one: cur < hi)
            item = 0;
            ++b;
            enter(p);
          }
          cost = span(p, b, item);
        }
      }
      if (j1 > 0) return true;
    }
  }
};

// log2 of a scale, exact for powers of two; -inf for zero, NaN below it.
__device__ __forceinline__ float log2_scale(float v) {
  int e;
  const float m = frexpf(v, &e);
  return m == 0.5f ? static_cast<float>(e - 1) : static_cast<float>(e) + __log2f(m);
}

// Sixteen e4m3 values to fp16, exactly.
__device__ __forceinline__ void widen16(const uint4& x, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(r[2 * i]), "=r"(r[2 * i + 1])
        : "r"(w[i]));
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// Four consecutive columns of tensor memory.
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, float* v) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, float* v) {
  if constexpr (N % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 16) tmem_ld16(taddr + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) tmem_ld4(taddr + i, v + i);
  }
}

// Eight or sixteen columns of tensor memory, written.
template <int N>
__device__ __forceinline__ void tmem_stn(uint32_t taddr, const uint32_t* v) {
  static_assert(N == 8 || N == 16, "columns");
  if constexpr (N == 16) {
    tmem_st16u(taddr, v);
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  }
}

// A barrier of the softmax warps, and one that says whether `bad` is set in any of their threads.
template <int THREADS>
__device__ __forceinline__ void softmax_sync() {
  asm volatile("barrier.cta.sync 1, %0;" ::"n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ bool softmax_any(bool bad) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(bad)), "n"(THREADS)
      : "memory");
  return r != 0u;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// A bounded wait of few instructions: a number of suspended looks of up to 20 us each, after which the
// site is left in `failed` for the CTA's end to report, and every later wait gives up at once.
constexpr uint32_t EXTEND_LOOKS = 1u << 17;
__device__ __forceinline__ bool extend_wait(uint32_t bar, uint32_t parity, volatile int* failed, int site) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < EXTEND_LOOKS; ++i) {
    if (mbar_try_wait_sleep(bar, parity, DU_WAIT_SLEEP_NS)) return true;
    if (*failed) return false;
  }
  *failed = site;
  return false;
}

template <int D, int NT, int CP>
__global__ void __launch_bounds__(EXTEND_THREADS, 1) extend_paged_kernel(const ExtendPagedParams p) {
  using S = ExtendShape<D, NT, CP>;
  constexpr int KT = S::KT, RP = S::RP, SPAN = S::SPAN, GPT = S::GPT, NB = S::NB, NS = S::NS, RPT = S::RPT;
  constexpr bool ALT = S::ALT;
  constexpr int NK = S::NK, NV = S::NV, NRK = S::NRK, NRV = S::NRV, NF = S::NF;
  constexpr uint32_t SWZ = swizzle_code(SPAN);
  constexpr uint32_t IDESC_QK = idesc_f16(128, KT, 0, 0, 0, 0);
  constexpr uint32_t IDESC_PV = idesc_f16(128, D, 0, 0, 0, 1);

  // The place of a stream's n-th tile of S, and the parity of its barriers.
  auto place = [](int n) { return S::SB == 2 ? n & 1 : 0; };
  auto turn = [](int n) { return S::SB == 2 ? (n >> 1) & 1 : n & 1; };
  // With one tile of S, P V begins with half of P. The products of one thread are known to complete in order if
  // they are of one shape; else the end of P V is waited for before its P is overwritten by a later S.
  constexpr bool HALVES = S::SB == 1 && CP == 1, ORDERED = S::SB == 1 && D == KT;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t sbase = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw_u32);
  auto bar = [&](int i) -> uint32_t { return sbase + S::OFF_BAR + 8u * static_cast<uint32_t>(i); };
  auto RKF = [&](int s) { return bar(S::B_RKF + s); };  // cached piece of K landed
  auto RKE = [&](int s) { return bar(S::B_RKE + s); };  // and widened
  auto RVF = [&](int s) { return bar(S::B_RVF + s); };
  auto RVE = [&](int s) { return bar(S::B_RVE + s); };
  auto KF = [&](int s) { return bar(S::B_KF + s); };    // widened K written
  auto KE = [&](int s) { return bar(S::B_KE + s); };    // and multiplied, by each stream that has it
  auto VF = [&](int s) { return bar(S::B_VF + s); };
  auto VE = [&](int s) { return bar(S::B_VE + s); };
  auto SCF = [&](int s) { return bar(S::B_SCF + s); };  // batch of scales written
  auto SCE = [&](int s) { return bar(S::B_SCE + s); };  // read by the softmax warps and those that widen V
  auto QF = [&](int x) { return bar(S::B_QF + x); };    // query rows written
  auto SF = [&](int x, int i) { return bar(S::B_SF + 2 * x + i); };  // S of stream x complete, in place i
  auto PF = [&](int x, int i) { return bar(S::B_PF + 2 * x + i); };  // P written, in place i (HALVES: its i-th half)
  auto OD = [&](int x) { return bar(S::B_OD + x); };    // P V of a tile done
  auto OF = [&](int x) { return bar(S::B_OF + x); };    // O of stream x final
  auto FF = [&](int i) { return bar(S::B_FF + i); };    // fragment entry written
  auto FE = [&](int i) { return bar(S::B_FE + i); };    // and read by every warp that takes it
  auto DR = [&](int i) { return bar(S::B_DR + i); };    // all products of an issuing warp done

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(sgen + S::OFF_WORDS);
  volatile int* failed = reinterpret_cast<volatile int*>(sgen + S::OFF_WORDS + 4);
  volatile int* frags = reinterpret_cast<volatile int*>(sgen + S::OFF_FRAG);

  if (tid == 0) {
    for (int s = 0; s < NRK; ++s) {
      mbar_init(RKF(s), 1);
      mbar_init(RKE(s), S::WC);
    }
    for (int s = 0; s < NRV; ++s) {
      mbar_init(RVF(s), 1);
      mbar_init(RVE(s), S::WC);
    }
    for (int s = 0; s < NK; ++s) {
      mbar_init(KF(s), S::WC);
      mbar_init(KE(s), NT);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(VF(s), S::WC);
      mbar_init(VE(s), NT);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(SCF(s), 1);
      mbar_init(SCE(s), S::SW + S::WC);
      mbar_init(QF(s), ALT ? 8 : 4);
      for (int i = 0; i < 2; ++i) {
        mbar_init(SF(s, i), 1);
        mbar_init(PF(s, i), 4);
      }
      mbar_init(OD(s), 1);
      mbar_init(OF(s), 1);
      mbar_init(DR(s), 1);
    }
    for (int s = 0; s < NF; ++s) {
      mbar_init(FF(s), 1);
      mbar_init(FE(s), S::SW + 2 * S::WC + 1 + NS);
    }
    *failed = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  griddep_wait();
  fence_proxy_async_global();  // (the caches are read by bulk copies)
  if (warp == 14) {
    tmem_alloc(sbase + S::OFF_WORDS, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The next fragment; kind 0: there is none, -1: a wait expired.
  int n_frag = 0;
  auto take = [&]() -> ExtendFrag {
    ExtendFrag f;
    const int s = n_frag % NF;
    const bool ok = __all_sync(0xffffffffu, extend_wait(FF(s), (n_frag / NF) & 1, failed, 500));
    const volatile int* e = frags + 16 * s;
    f.kind = ok ? e[0] : -1;
    f.b = e[1];
    f.kvh = e[2];
    f.row0 = e[3];
    f.rows = e[4];
    f.past = e[5];
    f.len = e[6];
    f.j0 = e[7];
    f.j1 = e[8];
    f.nk0 = e[9];
    f.nk1 = e[10];
    f.nf = e[11];
    f.c0 = e[12];
    f.slot = e[13];
    __syncwarp();
    if (lane == 0) mbar_arrive(FE(s));
    ++n_frag;
    return f;
  };
  // Key tiles of a fragment that stream x has.
  auto tiles_of = [&](const ExtendFrag& f, int x) -> int {
    const int nt = f.j1 - f.j0;
    if (ALT) return (nt - x + 1) >> 1;
    return max(0, min(f.j1, x ? f.nk1 : f.nk0) - f.j0);
  };

  if (warp < S::SW) {
    // ------------------------------------------------------------------ softmax
    regs_inc<S::REG_SOFTMAX>();
    const int x = warp >> 2, w4 = warp & 3;  // stream
    const int xr = ALT ? 0 : x;              // row tile
    const int row = 32 * w4 + lane;          // row of the tile = TMEM lane
    const int part = w4 / S::RW;             // the copy that the row belongs to
    const uint32_t lane_off = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t q_tile = sbase + S::OFF_Q + xr * S::Q_BYTES;
    const uint32_t s_addr0 = tmem + lane_off + S::TM_S + S::SB * x * KT, o_addr = tmem + lane_off + S::TM_O + x * D;
    constexpr int ST = 32 * S::SW;           // softmax threads
    int n_tile = 0, n_batch = 0, n_of = 0;
    while (true) {
      const ExtendFrag f = take();
      if (f.kind <= 0) {
        if (S::PARTS > 1) softmax_any<ST>(f.kind < 0);
        break;
      }
      const int nt = f.j1 - f.j0, n = tiles_of(f, x);
      const int r_item = CP > 1 ? row % (128 / CP) : xr * 128 + row;   // row of the item
      const bool row_ok = r_item < f.rows;
      const int r_all = f.row0 + min(r_item, f.rows - 1);
      const int t = small_div(r_all, p.G);                             // its token and head
      const int h = f.kvh * p.G + (r_all - t * p.G);
      const long long q_row = (static_cast<long long>(f.b) * p.Hq + h) * p.T + t;
      const int kmax = f.past + t;                                     // the last key that it sees
      const int kmin = f.past + small_div(f.row0 + min(xr * 128, f.rows - 1), p.G);  // that every row of the tile sees
      const bool warp_rows = r_item - lane < f.rows;                   // some row of the warp is one
      float qs = 0.f;  // the row's factor
      bool ok = true;
      if (ALT || n > 0) {
        // The warp's query rows: rotated in fp32, times a power of two (of each row) that brings its largest input
        // to [2^8, 2^9), as fp16. LPR lanes share a row, each with a pair of 16-byte pieces at a time: a row per
        // lane would touch 32 lines with each load, 4 us for 256 rows. First the rows as they are, where they
        // belong, and the largest of each; then the rotation in place. Streams that share the rows take turns.
        constexpr int LPR = D / 16, RPS = 32 / LPR;
        constexpr int UN = LPR < 8 ? LPR : 8;  // steps in flight
        const int piece = lane % LPR, in_step = lane / LPR;
        const int steps = min(LPR, (f.rows - (r_item - lane) + RPS - 1) / RPS);  // that have rows
        if (warp_rows) {
          const uint8_t* cp = static_cast<const uint8_t*>(p.cos) + static_cast<long long>(kmax) * D;
          const uint8_t* sp = static_cast<const uint8_t*>(p.sin) + static_cast<long long>(kmax) * D;
          for (int i = 0; i < D; i += 128) {
            prefetch_l1(cp + i);
            prefetch_l1(sp + i);
          }
          uint32_t top = 0u;
          const int q_row_lo = static_cast<int>(q_row), q_row_hi = static_cast<int>(q_row >> 32);
          auto row_of = [&](int from) {
            return static_cast<long long>(__shfl_sync(0xffffffffu, q_row_hi, from)) << 32 | static_cast<uint32_t>(__shfl_sync(0xffffffffu, q_row_lo, from));
          };
#pragma unroll 1
          for (int s0 = 0; s0 < steps; s0 += UN) {
            uint4 a[UN], b[UN];
#pragma unroll
            for (int i = 0; i < UN; ++i) {
              const uint8_t* src = static_cast<const uint8_t*>(p.q) + row_of((s0 + i) * RPS + in_step) * (2 * D) + 16 * piece;
              a[i] = ldg_v4(src);
              b[i] = ldg_v4(src + D);
            }
#pragma unroll
            for (int i = 0; i < UN; ++i) {
              const int at = 32 * w4 + (s0 + i) * RPS + in_step;
              if (!ALT || (i & 1) == x) {  // (s0 is even, or 0)
                st_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, at, piece), a[i]);
                st_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, at, piece + LPR), b[i]);
              }
              uint32_t big = 0u;
              const uint32_t w[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
              for (int k = 0; k < 8; ++k) big = __vmaxu2(big, w[k] & 0x7fff7fffu);
#pragma unroll
              for (int o = 1; o < LPR; o <<= 1) big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, o));
              big = __shfl_sync(0xffffffffu, big, lane % RPS * LPR);
              if (lane / RPS == s0 + i) top = big;
            }
          }
          const float2 tops = p.bf16 ? split2<true>(top) : split2<false>(top);
          const uint32_t top_bits = __float_as_uint(fmaxf(tops.x, tops.y));
          int e = static_cast<int>(top_bits >> 23) - 127;
          if (e == -127 || e == 128) e = 8;  // (zero, or not finite)
          e = min(max(e - 8, -100), 100);
          const float up_own = __int_as_float((127 - e) << 23);
          qs = __int_as_float((127 + e) << 23);
          __syncwarp();
          auto rotate = [&](auto bf16) {
            constexpr bool BF = decltype(bf16)::value;
            constexpr int TURN = ALT ? 2 : 1, PL = LPR < 2 * TURN ? 1 : 2;  // (more at a time would be code fetched once)
#pragma unroll 1
            for (int s0 = ALT ? x : 0; s0 < steps; s0 += TURN * PL) {
              uint4 a[PL], b[PL], c[PL], s[PL];
              uint32_t lo_at[PL], hi_at[PL];
              float up[PL];
#pragma unroll
              for (int i = 0; i < PL; ++i) {
                const int from = (s0 + i * TURN) * RPS + in_step, at = 32 * w4 + from;  // (rows past the last step's: below 32)
                up[i] = __shfl_sync(0xffffffffu, up_own, from);
                const int pos = __shfl_sync(0xffffffffu, kmax, from);
                lo_at[i] = q_tile + swz_chunk_offset<SPAN>(128, at, piece);
                hi_at[i] = q_tile + swz_chunk_offset<SPAN>(128, at, piece + LPR);
                a[i] = ld_shared_v4(lo_at[i]);
                b[i] = ld_shared_v4(hi_at[i]);
                c[i] = ldg_v4(static_cast<const uint8_t*>(p.cos) + static_cast<long long>(pos) * D + 16 * piece);
                s[i] = ldg_v4(static_cast<const uint8_t*>(p.sin) + static_cast<long long>(pos) * D + 16 * piece);
              }
#pragma unroll
              for (int i = 0; i < PL; ++i) {
                const uint32_t aa[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, ba[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
                const uint32_t ca[4] = {c[i].x, c[i].y, c[i].z, c[i].w}, sa[4] = {s[i].x, s[i].y, s[i].z, s[i].w};
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint64_t U = f2(up[i], up[i]), C = widen2<BF>(ca[k]), N = widen2<BF>(sa[k]);
                  const uint64_t A = f2_mul(widen2<BF>(aa[k]), U), B = f2_mul(widen2<BF>(ba[k]), U);
                  const float2 l2 = f2_split(f2_fma(B, f2_mul(N, f2(-1.f, -1.f)), f2_mul(A, C))), h2 = f2_split(f2_fma(A, N, f2_mul(B, C)));
                  lo[k] = pack2<false>(l2.x, l2.y);
                  hi[k] = pack2<false>(h2.x, h2.y);
                }
                st_shared_v4(lo_at[i], make_uint4(lo[0], lo[1], lo[2], lo[3]));
                st_shared_v4(hi_at[i], make_uint4(hi[0], hi[1], hi[2], hi[3]));
              }
            }
          };
          if (p.bf16) rotate(std::true_type{});
          else rotate(std::false_type{});
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(QF(xr));
      }
      // The reference of the weights is m + mlo (log2 domain); mlo is 0 but for references so large that
      // a sum with log2 vs would round away. l: the sum of 2^(s + vr - m - mlo + 8), with `far` of
      // 2^(s - m - eo).
      float m = -INFINITY, mlo = 0.f, l = 0.f, eo = -INFINITY, vr = 0.f;
      bool far = false;
      for (int jj = 0; jj < nt; ++jj) {
        const int bs = n_batch & 1;
        const uint8_t* sc = sgen + S::OFF_SC + bs * S::SC_BYTES;
        if (jj % NB == 0) {
          ok = __all_sync(0xffffffffu, extend_wait(SCF(bs), (n_batch >> 1) & 1, failed, 502));
          if (!ok) break;
          const bool now = *reinterpret_cast<const int*>(sc + 384 + 4 * NB + 4) != 0;
          if (jj == 0) vr = *reinterpret_cast<const float*>(sc + 384 + 4 * NB);
          if (now && !far) {
            far = true;
            eo = l == 0.f ? -INFINITY : mlo - EXTEND_TOP - vr;
          }
        }
        if (ALT ? (jj & 1) == x : jj < n) {
          ok = __all_sync(0xffffffffu, extend_wait(SF(x, place(n_tile)), turn(n_tile), failed, 503));
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_addr = s_addr0 + place(n_tile) * KT;
          const bool first = ALT ? jj < 2 : jj == 0;                 // this stream has no O yet
          const int lim = kmax - (f.j0 + jj) * KT - part * S::KC;    // columns beyond it are hidden from this row
          const bool diag = (f.j0 + jj) * KT + KT - 1 > kmin;        // some key of the tile is hidden from some row
          const float* scq = reinterpret_cast<const float*>(sc) + (jj % NB) * GPT + part * (S::KC / 16);  // (log2 vs 32 words behind, factors 64)
          if (warp_rows) {
            // S in two halves: the first is reduced while the second loads.
            constexpr int KC = S::KC, HALF = KC / 2, NG = KC / 16, GS = NG < 2 ? 1 : 2;
            float s[KC], kq[NG], ga[NG];
            tmem_ldn<HALF>(s_addr + part * KC, s);
#pragma unroll
            for (int g = 0; g < NG; ++g) kq[g] = scq[g] * qs;
            float mx = -INFINITY;
#pragma unroll
            for (int c0 = 0; c0 < KC; c0 += HALF) {
              tmem_wait_ld();
              if (c0 == 0) tmem_ldn<HALF>(s_addr + part * KC + HALF, s + HALF);
              if (__builtin_expect(diag, 0)) {
                // Hidden keys have a score of -inf, and where a whole group is hidden its scales do not count.
#pragma unroll
                for (int c = c0; c < c0 + HALF; ++c)
                  if (c > lim) s[c] = -INFINITY;
#pragma unroll
                for (int g = c0 / 16; g < (c0 + HALF) / 16; ++g)
                  if (kq[g] == 0.f || 16 * g > lim) kq[g] = FLT_MIN;  // (times -inf it has to be -inf)
              }
#pragma unroll
              for (int g = c0 / 16; g < (c0 + HALF) / 16; ++g) {
                float a = fmaxf(s[16 * g], s[16 * g + 1]), b = fmaxf(s[16 * g + 2], s[16 * g + 3]);
#pragma unroll
                for (int c = 16 * g + 4; c < 16 * g + 16; c += 4) {
                  a = max3(a, s[c], s[c + 1]);
                  b = max3(b, s[c + 2], s[c + 3]);
                }
                ga[g] = fmaxf(a, b);
                mx = fmaxf(mx, fmaf(ga[g], kq[g], scq[32 + g]));
              }
            }
            // (a row that is not there has whatever shared memory held, and no say in what its warp does)
            if (!row_ok) mx = -INFINITY;
            const float m_old = m, mlo_old = mlo;
            bool moved = mx > m + mlo + EXTEND_MOVE;
            float base = 0.f;  // what is taken off log2 vs
            // (infinities: a row without keys so far, or one that will be NaN)
            const bool large = (fabsf(m) > EXTEND_LARGE && fabsf(m) < INFINITY) || (fabsf(mx) > EXTEND_LARGE && fabsf(mx) < INFINITY);
            const bool any = far || __any_sync(0xffffffffu, moved || large);
            if (__builtin_expect(!any || (!far && !__any_sync(0xffffffffu, large)), 1)) {
              if (moved) {
                m = mx;
                mlo = 0.f;
              }
              if (m != -INFINITY) base = m + mlo;
            } else {
              // Scores relative to the reference first, then the rest: nothing is rounded away beside a
              // large score. The product is rounded before the reference is taken off, so that scores that are
              // alike have the same weight whatever their size.
              auto less = [](float a, float k, float r) { return __fadd_rn(__fmul_rn(a, k), -r); };
              float hi = -INFINITY, lo = -INFINITY;
#pragma unroll
              for (int g = 0; g < NG; ++g) hi = fmaxf(hi, ga[g] * kq[g]);
              if (!row_ok) hi = -INFINITY;
              const float h0 = hi == -INFINITY ? 0.f : hi;
#pragma unroll
              for (int g = 0; g < NG; ++g) lo = fmaxf(lo, less(ga[g], kq[g], h0) + scq[32 + g]);
              moved = m == -INFINITY ? hi != -INFINITY : (hi - m) + (lo - mlo) > EXTEND_MOVE;
              if (moved) {
                m = hi;
                mlo = lo;
              }
              const float mr = m == -INFINITY ? 0.f : m;
              base = m == -INFINITY ? 0.f : mlo;
#pragma unroll
              for (int c = 0; c < KC; ++c) s[c] = less(s[c], kq[c / 16], mr);
#pragma unroll
              for (int g = 0; g < NG; ++g) kq[g] = 1.f;
              if (far) {
                // Value scales far apart: the sum has a reference of its own, eo beyond m.
                if (moved && m_old != -INFINITY) eo += m_old - m;
                const float en = fmaxf(l == 0.f ? -INFINITY : eo, hi == -INFINITY ? -INFINITY : hi - mr);
                const float e0 = en == -INFINITY ? 0.f : en;
                l = l == 0.f ? 0.f : l * ex2(eo - e0);
                eo = en;
#pragma unroll
                for (int c = 0; c < KC; ++c) l += ex2(s[c] - e0);
              }
            }
            if (__builtin_expect(any && !first && __any_sync(0xffffffffu, moved), 0)) {
              // (O has to have the products of the tile before; the one tile of S is there after them)
              if (S::SB == 2) {
                ok = __all_sync(0xffffffffu, extend_wait(OD(x), (n_tile - 1) & 1, failed, 504));
                tc_fence_after();
              }
              const float alpha = moved && m_old != -INFINITY ? ex2((m_old - m) + (mlo_old - mlo)) : 1.0f;
              if (!far) l *= alpha;
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                tmem_ld16(o_addr + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] *= alpha;
                tmem_st16(o_addr + c, o);
              }
            }
            if constexpr (CP > 1) {  // nothing for the keys of the other copies
              constexpr int W = KC / 2 < 16 ? KC / 2 : 16;
              const uint32_t none[W] = {};
#pragma unroll
              for (int c = 0; c < KT / 2; c += W)
                if (c / (KC / 2) != part) tmem_stn<W>(s_addr + c, none);
            }
            uint64_t acc = f2(0.f, 0.f);
#pragma unroll
            for (int g = 0; g < NG; g += GS) {
              uint32_t pk[8 * GS];
#pragma unroll
              for (int q = g; q < g + GS; ++q) {
                // (a group that is hidden from the row has scores of -inf, whatever its scales)
                float lv = scq[32 + q], iv = scq[64 + q];
                if (__builtin_expect(diag, 0) && 16 * q > lim) {
                  lv = vr;
                  iv = 1.f;
                }
                const float add = lv - base + EXTEND_TOP;
                const uint64_t A = f2(add, add), K = f2(kq[q], kq[q]);
                uint64_t sum = f2(0.f, 0.f);
#pragma unroll
                for (int c = 16 * q; c < 16 * q + 16; c += 2) {
                  const float2 xx = f2_split(f2_fma(f2(s[c], s[c + 1]), K, A));
                  const float2 pp = make_float2(ex2(xx.x), ex2(xx.y));
                  sum = f2_add(sum, f2(pp.x, pp.y));
                  pk[c / 2 - 8 * g] = pack2<false>(pp.x, pp.y);
                }
                acc = f2_fma(sum, f2(iv, iv), acc);
              }
              tmem_stn<8 * GS>(s_addr + part * (KC / 2) + 8 * g, pk);
              if (HALVES && g + 2 == NG / 2) {
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(PF(x, 0));
              }
            }
            if (!far) {
              const float2 rs = f2_split(acc);
              l += rs.x + rs.y;
            }
            tmem_wait_st();
          } else if (HALVES && lane == 0) {
            mbar_arrive(PF(x, 0));
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(PF(x, HALVES ? 1 : place(n_tile)));
          ++n_tile;
          if (!ok) break;
        }
        if (jj % NB == NB - 1 || jj == nt - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(SCE(bs));
          ++n_batch;
        }
      }
      if (ok && n > 0) ok = __all_sync(0xffffffffu, extend_wait(OF(x), n_of++ & 1, failed, 505));
      // Where a row has parts, every softmax warp comes here once per fragment, whatever happened to it, and all
      // go on or none. Else each goes its own way (the others' waits expire with its own).
      if (S::PARTS > 1 ? softmax_any<ST>(!ok) : !ok) break;
      tc_fence_after();
      // The log2 of the row's (or its part's) sum, in two parts; and what brings O to the fragment's output,
      // O 2^(m + mlo - 8) over the sum, in two factors since the exponent may be large. A sum that is not a number
      // (a block's scale, or a block without an id) must not look like no keys: the maximum passes over such scores.
      float2 lse = l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(l == l ? m : l, lg2(l) + (far ? eo : mlo - EXTEND_TOP - vr));
      float w1 = 0.f, w2 = 0.f;
      if (l != 0.f) {
        const float ex = far ? mlo - EXTEND_TOP - eo : vr, half = rintf(0.5f * ex);
        w2 = ex2(half);
        w1 = ex2(ex - half) / l;
      }
      // A row of a whole item sees a key at least. Where all that it sees have scores of -inf (an infinite query), its
      // softmax is not a number, as it is in an item that is cut, where the joining kernel divides by no weight.
      const bool whole = f.nf == 1;
      constexpr float not_a_number = __builtin_nanf("");
      float4* const part_o = reinterpret_cast<float4*>(p.part);
      float2* const part_l = reinterpret_cast<float2*>(p.part + 2LL * gridDim.x * RP * D);
      auto part_at = [&](int slot, int col, int r) { return (static_cast<long long>(slot) * (D / 4) + col / 4) * RP + r; };
      uint8_t* out = static_cast<uint8_t*>(p.out) + q_row * (2 * D);
      // N columns of the row (four or eight) from `col` on.
      auto pack4 = [&](const float* a) {
        return p.bf16 ? make_uint2(pack2<true>(a[0], a[1]), pack2<true>(a[2], a[3])) : make_uint2(pack2<false>(a[0], a[1]), pack2<false>(a[2], a[3]));
      };
      auto put = [&](int col, const auto& a) {
        constexpr int N = sizeof(a) / sizeof(float);
        if (f.nf > 1) {
#pragma unroll
          for (int i = 0; i < N; i += 4) part_o[part_at(f.slot, col + i, r_item)] = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
        } else {
          const uint2 u = pack4(a);
          if constexpr (N == 8) {
            const uint2 v = pack4(a + 4);
            *reinterpret_cast<uint4*>(out + 2 * col) = make_uint4(u.x, u.y, v.x, v.y);
          } else {
            *reinterpret_cast<uint2*>(out + 2 * col) = u;
          }
        }
      };
      if constexpr (CP > 1) {
        // The parts of a row joined: weights by their sums, then a quarter of the columns at a time, weighted,
        // through shared memory where the query rows were (a row's 16-byte pieces turned by the row's number). A
        // thread adds up its own row, of every so many columns.
        constexpr int PARTS = S::PARTS, ROWS = 128 / CP, CB = D / 4, PC = CB / 4, GROUPS = S::SW / S::RW;
        const int mine = (ALT ? x * CP : 0) + part;
        float2* lses = reinterpret_cast<float2*>(sgen + S::OFF_Q);
        float4* buf = reinterpret_cast<float4*>(sgen + S::OFF_Q);
        lses[mine * ROWS + r_item] = lse;
        softmax_sync<ST>();
        float2 top = make_float2(-INFINITY, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const float2 a = lses[i * ROWS + r_item];
          if (a.x == -INFINITY) continue;
          const float d = top.x == -INFINITY ? INFINITY : (a.x - top.x) + (a.y - top.y);
          const float e = ex2(-fabsf(d));
          sum = d > 0.f ? sum * e + 1.f : sum + e;  // (NaN where one is)
          if (d > 0.f || top.x == -INFINITY) top = a;
        }
        softmax_sync<ST>();
        if (lse.x != -INFINITY) w1 *= ex2((lse.x - top.x) + (lse.y - top.y)) / sum;
        if (top.x != -INFINITY) top.y += lg2(sum);
        else if (whole) w1 = not_a_number;
        if (f.nf > 1 && mine == 0 && row_ok) part_l[static_cast<long long>(f.slot) * RP + r_item] = top;
        // (two quarters, or all, where half or a quarter of the rows are there)
        const int at_once = f.rows > ROWS / 2 ? 1 : (f.rows > ROWS / 4 ? 2 : 4), rows_p = ROWS / at_once;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += at_once * CB) {
#pragma unroll 1
          for (int q = 0; q < at_once; ++q) {
            if (!warp_rows) continue;
            float o[CB];
            if (n > 0) {
              tmem_ldn<CB>(o_addr + c0 + q * CB, o);
              tmem_wait_ld();
            }
            if (row_ok) {
#pragma unroll
              for (int i = 0; i < PC; ++i)
                buf[((q * PARTS + mine) * rows_p + r_item) * PC + (i + r_item) % PC] =
                    n > 0 ? make_float4(o[4 * i] * w1 * w2, o[4 * i + 1] * w1 * w2, o[4 * i + 2] * w1 * w2, o[4 * i + 3] * w1 * w2) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
          softmax_sync<ST>();
          if (row_ok) {
#pragma unroll 1
            for (int c = mine; c < at_once * PC; c += GROUPS) {
              float a[4] = {};
#pragma unroll
              for (int i = 0; i < PARTS; ++i) {
                const float4 b = buf[((c / PC * PARTS + i) * rows_p + r_item) * PC + (c + r_item) % PC];
                a[0] += b.x;
                a[1] += b.y;
                a[2] += b.z;
                a[3] += b.w;
              }
              put(c0 + 4 * c, a);
            }
          }
          softmax_sync<ST>();
        }
      } else if constexpr (ALT) {
        // The two parts of a row joined: weights by their sums, then each stream finishes half of the columns,
        // a quarter of D at a time, the other's share of which comes through shared memory where the query
        // rows were (a row's 16-byte pieces turned by the row's number).
        float2* lses = reinterpret_cast<float2*>(sgen + S::OFF_Q);
        lses[x * 128 + row] = lse;
        softmax_sync<ST>();
        const float2 other = lses[(1 - x) * 128 + row];
        softmax_sync<ST>();
        if (other.x != -INFINITY) {
          if (lse.x == -INFINITY) {
            lse = other;
          } else {
            const float d = (other.x - lse.x) + (other.y - lse.y);  // (NaN where one is)
            const float e = ex2(-fabsf(d)), total = 1.f + e;
            w1 *= (d > 0.f ? e : 1.f) / total;
            if (d > 0.f) lse = other;
            lse.y += lg2(total);
          }
        }
        if (whole && lse.x == -INFINITY) w1 = not_a_number;
        if (f.nf > 1 && x == 0 && row_ok) part_l[static_cast<long long>(f.slot) * RP + row] = lse;
        constexpr int CB = D / 4, PC = CB / 4;
        float4* buf = reinterpret_cast<float4*>(sgen + S::OFF_Q);
        // `CB` of this stream's columns, weighted.
        auto mine = [&](int c0, float (&o)[CB]) {
          if (n > 0) {
            tmem_ldn<CB>(o_addr + c0, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < CB; ++i) o[i] = o[i] * w1 * w2;
          } else {
#pragma unroll
            for (int i = 0; i < CB; ++i) o[i] = 0.f;
          }
        };
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
          if (warp_rows) {
            float o[CB];
            mine((1 - x) * (D / 2) + pass * CB, o);
            if (row_ok) {
#pragma unroll
              for (int i = 0; i < PC; ++i) buf[((1 - x) * 128 + row) * PC + (i + row) % PC] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          }
          softmax_sync<ST>();
          if (warp_rows) {
            float o[CB];
            const int c0 = x * (D / 2) + pass * CB;
            mine(c0, o);
            if (row_ok) {
              constexpr int N = CB < 8 ? CB : 8;
#pragma unroll
              for (int c = 0; c < CB; c += N) {
                float a[N];
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                  const float4 b = buf[(x * 128 + row) * PC + ((c + i) / 4 + row) % PC];
                  a[i] = o[c + i] + b.x;
                  a[i + 1] = o[c + i + 1] + b.y;
                  a[i + 2] = o[c + i + 2] + b.z;
                  a[i + 3] = o[c + i + 3] + b.w;
                }
                put(c0 + c, a);
              }
            }
          }
          softmax_sync<ST>();
        }
      } else {
        if (f.nf > 1 && row_ok) part_l[static_cast<long long>(f.slot) * RP + r_item] = lse;
        if (whole && l == 0.f) w1 = not_a_number;
        if (n > 0 && warp_rows) {
          // Whole items' rows go out through shared memory, so that lanes share lines: each where its own query row
          // was, piece for piece. A warp so writes no bytes but those of its own query rows, which it is the next to
          // write, and no warp waits for the others; row after row, warps would share bytes from head_dim 128 on.
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_ld16(o_addr + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = o[i] * w1 * w2;
#pragma unroll
            for (int k = 0; k < 16; k += 8) {
              if (f.nf > 1) {
                if (row_ok) {
                  part_o[part_at(f.slot, c + k, r_item)] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                  part_o[part_at(f.slot, c + k + 4, r_item)] = make_float4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]);
                }
              } else {
                const uint2 u = pack4(o + k), v = pack4(o + k + 4);
                st_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, row, (c + k) / 8), make_uint4(u.x, u.y, v.x, v.y));
              }
            }
          }
          if (f.nf == 1) {
            constexpr int LPO = D / 8, RPO = 32 / LPO;  // lanes that share a row, rows of a step
            const int q_row_lo = static_cast<int>(q_row), q_row_hi = static_cast<int>(q_row >> 32);
            __syncwarp();
#pragma unroll 2
            for (int i = 0; i < LPO; ++i) {
              const int from = i * RPO + lane / LPO, at = 32 * w4 + from;
              const long long to = static_cast<long long>(__shfl_sync(0xffffffffu, q_row_hi, from)) << 32 |
                                   static_cast<uint32_t>(__shfl_sync(0xffffffffu, q_row_lo, from));
              const uint4 v = ld_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, at, lane % LPO));
              if (r_item - lane + from < f.rows) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + to * (2 * D) + 16 * (lane % LPO)) = v;
            }
            __syncwarp();
          }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ rows behind the last token
    regs_dec<S::REG_WIDEN>();
    {
      const int first = warp - S::SW;
      constexpr int warps = 12 - S::SW, P16 = D / 8;  // 16-byte pieces of a row
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        int n = p.T;
        if (b0 + lane < p.B) {
          int past, len;
          n = extend_new(p, b0 + lane, past, len);
          if (n < 0) {
            n = 0;
            if (blockIdx.x == 0 && first == 0) record_error(6u, static_cast<unsigned>(b0 + lane), static_cast<unsigned>(p.lens[b0 + lane]));
          }
        }
        for (unsigned todo = __ballot_sync(0xffffffffu, n < p.T); todo; todo &= todo - 1u) {
          const int l = __ffs(static_cast<int>(todo)) - 1, b = b0 + l;
          const int from = __shfl_sync(0xffffffffu, n, l);
          // every gridDim.x-th row set (b, h), each warp a share of its rows
          const unsigned g = gridDim.x, at = ((static_cast<unsigned>(b) % g) * (static_cast<unsigned>(p.Hq) % g)) % g;
          for (int h = static_cast<int>((blockIdx.x + g - at) % g); h < p.Hq; h += static_cast<int>(g)) {
            uint4* dst = reinterpret_cast<uint4*>(p.out) + ((static_cast<long long>(b) * p.Hq + h) * p.T + from) * P16;
            const long long pieces = static_cast<long long>(p.T - from) * P16;
            for (long long i = 32 * first + lane; i < pieces; i += 32 * warps) dst[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
    }
    // ------------------------------------------------------------------ widening
    const bool values = warp >= S::SW + S::WC;
    const int wt = (warp - S::SW) % S::WC * 32 + lane;  // thread of this cache's warps
    constexpr int CPR = D / 16;             // 16-byte parts of a cached row
    constexpr int PARTS = S::RK * CPR;      // of a copied piece
    constexpr int WT = PARTS < 32 * S::WC ? PARTS : 32 * S::WC;  // threads that have any
    constexpr int PER = PARTS / WT;
    // A thread's parts are RS rows apart, a multiple of the swizzle's period, so their offsets in the
    // widened tile are RS SPAN apart. Where a row has eight parts or more, a quarter-warp takes four of
    // one row and the next four of the row below: then neither its loads nor its stores meet in a bank.
    constexpr int RS = WT / CPR;
    static_assert(RS % 8 == 0 && PARTS % WT == 0, "a thread's parts");
    int r0 = wt / CPR, k0 = wt % CPR;
    if constexpr (CPR >= 8) {
      const int in = wt % (2 * CPR), below = (in >> 2) & 1;
      r0 = wt / (2 * CPR) * 2 + below;
      k0 = (in & 3) + 4 * ((in >> 3) ^ below);
    }
    const uint32_t from = 16 * (r0 * CPR + k0);
    const uint32_t to0 = swz_chunk_offset<SPAN>(KT, r0, 2 * k0), to1 = swz_chunk_offset<SPAN>(KT, r0, 2 * k0 + 1);
    const int n_raw = values ? NRV : NRK, n_wide = values ? NV : NK;
    const uint32_t raw0 = sbase + (values ? S::OFF_RV : S::OFF_RK) + from, wide0 = sbase + (values ? S::OFF_V : S::OFF_K);
    const uint32_t raw_full = values ? RVF(0) : RKF(0), raw_empty = values ? RVE(0) : RKE(0);
    const uint32_t wide_full = values ? VF(0) : KF(0), wide_empty = values ? VE(0) : KE(0);
    int rs = 0, rp = 0, ws = 0, wp = 1, n_batch = 0;  // stages and parities
    bool ok = true;
    while (ok) {
      const ExtendFrag f = take();
      if (f.kind <= 0) break;
      const int nt = f.j1 - f.j0;
      for (int jj = 0; ok && jj < nt; ++jj) {
        uint32_t zero = 0u;   // groups of V that are not to be used
        int rows_left = KT;   // rows up to the request's end
        if (values) {
          const int bs = n_batch & 1;
          if (jj % NB == 0) {
            ok = __all_sync(0xffffffffu, extend_wait(SCF(bs), (n_batch >> 1) & 1, failed, 510));
            if (!ok) break;
          }
          zero = *reinterpret_cast<const uint32_t*>(sgen + S::OFF_SC + bs * S::SC_BYTES + 384 + 4 * (jj % NB));
          rows_left = f.len - (f.j0 + jj) * KT;
          if (jj % NB == NB - 1 || jj == nt - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(SCE(bs));
            ++n_batch;
          }
        }
        ok = __all_sync(0xffffffffu, extend_wait(wide_empty + 8 * ws, wp, failed, 512));
        if (!ok) break;
        const bool clear = zero != 0u || (values && rows_left < KT);
        uint32_t dst = wide0 + ws * S::T_BYTES;
#pragma unroll 1
        for (int piece = 0; piece < RPT; ++piece) {
          ok = __all_sync(0xffffffffu, extend_wait(raw_full + 8 * rs, rp, failed, 511));
          if (!ok) break;
          if (WT == 32 * S::WC || wt < WT) {
            const uint32_t src = raw0 + rs * S::RAW;
            constexpr int UN = PER < 4 ? PER : 4;
#pragma unroll 1
            for (int i0 = 0; i0 < PER; i0 += UN) {
              uint4 b[UN];
#pragma unroll
              for (int i = 0; i < UN; ++i) b[i] = ld_shared_v4(src + 16 * RS * CPR * (i0 + i));
              if (__builtin_expect(clear, 0)) {
#pragma unroll
                for (int i = 0; i < UN; ++i) {
                  const int r = piece * S::RK + r0 + RS * (i0 + i);
                  if (r >= rows_left || ((zero >> (r / 16)) & 1u)) b[i] = make_uint4(0u, 0u, 0u, 0u);
                }
              }
#pragma unroll
              for (int i = 0; i < UN; ++i) {
                uint4 lo, hi;
                widen16(b[i], lo, hi);
                st_shared_v4(dst + to0 + RS * SPAN * (i0 + i), lo);
                st_shared_v4(dst + to1 + RS * SPAN * (i0 + i), hi);
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(raw_empty + 8 * rs);
          if (++rs == n_raw) {
            rs = 0;
            rp ^= 1;
          }
          dst += S::RK * SPAN;
        }
        if (!ok) break;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(wide_full + 8 * ws);
        if (++ws == n_wide) {
          ws = 0;
          wp ^= 1;
        }
      }
    }
  } else {
    regs_dec<S::REG_ISSUE>();
    const int keys = min(p.block, S::RK);        // of a copy
    const uint32_t bytes = static_cast<uint32_t>(keys) * D;
    constexpr int GPP = S::RK / 16;              // groups of 16 keys in a piece
    int st = 0, ph = 1, used = 0;                // a copying warp's stage, parity, stages that were used
    bool ok = true;
    // Up to eight pieces of a cache, of which a lane has the block id of a group of 16 keys from `key` on.
    auto copy = [&](const ExtendFrag& f, const uint8_t* cache, int id, int key, int pieces, int n_raw, uint32_t raw0, uint32_t full, uint32_t empty, int site) {
      const bool first = (16 * lane) % keys == 0 && static_cast<unsigned>(id) < static_cast<unsigned>(p.N);
      const uint8_t* src = cache + ((static_cast<long long>(id) * p.Hkv + f.kvh) * p.block + (key & (p.block - 1))) * D;
      const unsigned firsts = __ballot_sync(0xffffffffu, first);
#pragma unroll 1
      for (int i = 0; i < pieces; ++i) {
        ok = __all_sync(0xffffffffu, extend_wait(empty + 8 * st, ph, failed, site));
        if (!ok) break;
        const unsigned mine = firsts & (((1u << GPP) - 1u) << (i * GPP));
        if (lane == 0) mbar_expect_tx(full + 8 * st, __popc(mine) * bytes);
        __syncwarp();
        if ((mine >> lane) & 1u) bulk_load(raw0 + st * S::RAW + (lane % GPP) * 16 * D, src, bytes, full + 8 * st);
        used = max(used, st + 1);
        if (++st == n_raw) {
          st = 0;
          ph ^= 1;
        }
      }
    };
    if (warp == 12) {
      // ------------------------------------------------------------------ copies of K
      while (ok) {
        const ExtendFrag f = take();
        if (f.kind <= 0) break;
        const int np = (f.j1 - f.j0) * RPT, key0 = f.j0 * KT;
        const int* row = p.table + static_cast<long long>(f.b) * p.width;
        // A lane has a group of 16 keys of eight pieces; the ids of the next ones are fetched ahead.
        auto fetch = [&](int p0) {
          const int key = key0 + p0 * S::RK + 16 * lane;
          return key < f.len ? row[key >> p.block_log2] : -1;
        };
        int id = fetch(0);
        for (int p0 = 0; ok && p0 < np; p0 += 8) {
          const int next = p0 + 8 < np ? fetch(p0 + 8) : -1;
          copy(f, p.k8, id, key0 + p0 * S::RK + 16 * lane, min(8, np - p0), NRK, sbase + S::OFF_RK, RKF(0), RKE(0), 520);
          id = next;
        }
      }
      // Every copy lands before the CTA ends.
      for (int s = 0; s < used; ++s) mbar_wait_drain(RKF(s), static_cast<uint32_t>(s < st ? ph ^ 1 : ph), 521);
    } else if (warp >= 14 && warp < 14 + NS) {
      // ------------------------------------------------------------------ products of stream x
      const int x = warp - 14;
      const uint64_t dq = smem_desc(sbase + S::OFF_Q + (ALT ? 0 : x) * S::Q_BYTES, 16, 8 * SPAN, SWZ);
      const uint64_t dk0 = smem_desc(sbase + S::OFF_K, 16, 8 * SPAN, SWZ);
      const uint64_t dv0 = smem_desc(sbase + S::OFF_V, KT * SPAN, 8 * SPAN, SWZ);
      const uint32_t s_tmem = tmem + S::TM_S + S::SB * x * KT, o_tmem = tmem + S::TM_O + x * D;
      const bool leader = elect_one();
      int kt = 0;                        // key tiles of the fragments before
      int n_q = 0, n_s = 0, n_p = 0;     // query tiles, tiles of S and of P
      auto wait = [&](uint32_t b, int parity, int site) {
        return __all_sync(0xffffffffu, extend_wait(b, parity, failed, site)) != 0;
      };
      // S of tile jj of the fragment, once its widened K is there.
      auto scores = [&](int jj) {
        const int st = (kt + jj) % NK;
        if (!(ok = wait(KF(st), ((kt + jj) / NK) & 1, 533))) return;
        tc_fence_after();
        if (leader) {
          const uint64_t dk = dk0 + static_cast<uint64_t>((st * S::T_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off_q = ((kk * 32) / SPAN) * 128 * SPAN + (kk * 32) % SPAN;
            const uint32_t off_k = ((kk * 32) / SPAN) * KT * SPAN + (kk * 32) % SPAN;
            umma_f16_ss(s_tmem + place(n_s) * KT, dq + (off_q >> 4), dk + (off_k >> 4), IDESC_QK, kk > 0 ? 1u : 0u);
          }
          umma_commit(SF(x, place(n_s)));
          umma_commit(KE(st));
        }
        __syncwarp();
        ++n_s;
      };
      while (ok) {
        const ExtendFrag f = take();
        if (f.kind <= 0) break;
        const int nt = f.j1 - f.j0, n = tiles_of(f, x);
        const int step = ALT ? 2 : 1, first = ALT ? x : 0;
        if (ALT || n > 0) ok = wait(QF(ALT ? 0 : x), n_q++ & 1, 530);
        if (ok && n > 0) scores(first);
        if (S::SB == 2 && ok && n > 1) scores(first + step);
        for (int i = 0; ok && i < n; ++i) {
          const int jj = first + i * step, st = (kt + jj) % NV;
          if (!(ok = wait(VF(st), ((kt + jj) / NV) & 1, 532))) break;
          const uint64_t dv = dv0 + static_cast<uint64_t>((st * S::T_BYTES) >> 4);
          constexpr int PH = HALVES ? 2 : 1;
#pragma unroll
          for (int half = 0; half < PH; ++half) {
            if (!(ok = wait(PF(x, HALVES ? half : place(n_p)), turn(n_p), 531))) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int kk = half * (KT / 16 / PH); kk < (half + 1) * (KT / 16 / PH); ++kk)
                umma_f16_ts(o_tmem, s_tmem + place(n_p) * KT + kk * 8, dv + static_cast<uint64_t>((kk * 16 * SPAN) >> 4), IDESC_PV, (i > 0 || kk > 0) ? 1u : 0u);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (leader) {
            umma_commit(VE(st));
            if (!ORDERED) umma_commit(OD(x));
            if (i == n - 1) umma_commit(OF(x));
          }
          __syncwarp();
          // The next S (but one, with two) overwrites this P.
          if (i + S::SB < n) {
            if (!ORDERED && !(ok = wait(OD(x), n_p & 1, 534))) break;
            scores(jj + S::SB * step);
          }
          ++n_p;
        }
        if (NT == 2) {
          // Tiles that only the other stream has: released as they come.
          for (int jj = n; ok && jj < nt; ++jj) {
            const int st = (kt + jj) % NK, sv = (kt + jj) % NV;
            if (!(ok = wait(KF(st), ((kt + jj) / NK) & 1, 537))) break;
            if (lane == 0) mbar_arrive(KE(st));
            if (!(ok = wait(VF(sv), ((kt + jj) / NV) & 1, 538))) break;
            if (lane == 0) mbar_arrive(VE(sv));
          }
        }
        kt += nt;
      }
      // Every product is done before tensor memory is released.
      if (leader) {
        umma_commit(DR(x));
        mbar_wait_drain(DR(x), 0, 535);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ------------------------------------------------------------------ fragments, scales, copies of V
      ExtendWalk<S> walk;
      walk.init(p, lane);
      int* split = p.split + 8 * blockIdx.x;
      if (lane == 0) split[0] = 0;
      int nfr = 0, n_batch = 0;
      while (true) {
        ExtendFrag f{};
        const bool more = walk.next(p, f);
        if (!more) f.kind = 0;
        const int slot = nfr % NF;
        if (nfr >= NF) ok = __all_sync(0xffffffffu, extend_wait(FE(slot), (nfr / NF - 1) & 1, failed, 540));
        if (!ok) break;
        if (lane == 0) {
          volatile int* e = frags + 16 * slot;
          e[0] = f.kind;
          e[1] = f.b;
          e[2] = f.kvh;
          e[3] = f.row0;
          e[4] = f.rows;
          e[5] = f.past;
          e[6] = f.len;
          e[7] = f.j0;
          e[8] = f.j1;
          e[9] = f.nk0;
          e[10] = f.nk1;
          e[11] = f.nf;
          e[12] = f.c0;
          e[13] = f.slot;
          mbar_arrive(FF(slot));
          if (more && f.nf > 1 && f.j0 == 0) {
            split[1] = f.b;
            split[2] = f.kvh;
            split[3] = f.row0;
            split[4] = f.rows;
            split[0] = f.nf;
          }
        }
        __syncwarp();
        ++nfr;
        if (!more) break;
        // The query rows on their way into L2 (the softmax gets to them a fragment later).
        for (int r = lane; r < f.rows; r += 32) {
          const int t = small_div(f.row0 + r, p.G), h = f.kvh * p.G + (f.row0 + r - t * p.G);
          const uint8_t* src = static_cast<const uint8_t*>(p.q) + ((static_cast<long long>(f.b) * p.Hq + h) * p.T + t) * (2 * D);
#pragma unroll 1
          for (int i = 0; i < 2 * D; i += 128) prefetch_l2(src + i);
        }
        const int nt = f.j1 - f.j0;
        const int* row = p.table + static_cast<long long>(f.b) * p.width;
        float vr = 0.f;
        bool far = false;
        // A lane has a group of 16 keys of NB tiles; the ids and scales of the next ones are fetched ahead.
        int id = -1;
        float ks = 0.f, vs = 1.f;
        bool live = false;
        auto fetch = [&](int t0) {
          const int key = (f.j0 + t0) * KT + 16 * lane;
          live = key < f.len && key < f.j1 * KT;
          ks = 0.f;
          vs = 1.f;
          id = -1;
          if (live) {
            id = row[key >> p.block_log2];
            if (static_cast<unsigned>(id) < static_cast<unsigned>(p.N)) {
              const long long cell = static_cast<long long>(id) * p.Hkv + f.kvh;
              ks = p.ks[cell];
              vs = p.vs[cell];
            }
          }
        };
        fetch(0);
        for (int t0 = 0; t0 < nt; t0 += NB) {
          const bool good = !live || static_cast<unsigned>(id) < static_cast<unsigned>(p.N);
          if (!good) record_error(7u, static_cast<unsigned>(f.b), static_cast<unsigned>(id));
          ks = good ? ks * p.scale_log2 : __int_as_float(0x7fc00000);
          float lv = log2_scale(vs);
          if (t0 == 0) {
            vr = __shfl_sync(0xffffffffu, lv, 0);
            if (!(fabsf(vr) < 200.f)) vr = 0.f;
          }
          if (!live || !good) lv = vr;
          const bool nan = lv != lv;
          const float d = vr - lv;
          far = far || __any_sync(0xffffffffu, fabsf(d) > EXTEND_FAR);
          const unsigned bad = __ballot_sync(0xffffffffu, !good || nan || ks != ks);
          const int bs = n_batch & 1;
          if (n_batch >= 2) ok = __all_sync(0xffffffffu, extend_wait(SCE(bs), ((n_batch >> 1) - 1) & 1, failed, 541));
          if (!ok) break;
          uint8_t* sc = sgen + S::OFF_SC + bs * S::SC_BYTES;
          reinterpret_cast<float*>(sc)[lane] = ks;
          reinterpret_cast<float*>(sc + 128)[lane] = lv;
          reinterpret_cast<float*>(sc + 256)[lane] = nan ? 1.f : exp2f(d);
          if (lane < NB) reinterpret_cast<uint32_t*>(sc + 384)[lane] = (bad >> (lane * GPT)) & ((1u << GPT) - 1u);
          if (lane == 0) {
            *reinterpret_cast<float*>(sc + 384 + 4 * NB) = vr;
            *reinterpret_cast<int*>(sc + 384 + 4 * NB + 4) = far;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(SCF(bs));
          ++n_batch;
          const int at = id, key = (f.j0 + t0) * KT + 16 * lane;
          if (t0 + NB < nt) fetch(t0 + NB);
          copy(f, p.v8, at, key, min(8, (nt - t0) * RPT), NRV, sbase + S::OFF_RV, RVF(0), RVE(0), 522);
          if (!ok) break;
        }
        if (!ok) break;
      }
      for (int s = 0; s < used; ++s) mbar_wait_drain(RVF(s), static_cast<uint32_t>(s < st ? ph ^ 1 : ph), 523);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 14) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
  if (tid == 0 && *failed) record_timeout(static_cast<unsigned>(*failed));
}

// Joins the fragments of items that lie across CTAs. Block (c, k) takes the k-th share of the item that CTA c
// of the kernel before has the first fragment of, if it has one: a thread has a row, and eight columns of it.
// Bound by the partials' reads from L2 (and, where there are none, by the launch).
constexpr int EXTEND_JOIN_THREADS = 256;
template <int D, int NT>
__global__ void __launch_bounds__(EXTEND_JOIN_THREADS) extend_join_kernel(const ExtendPagedParams p, int ctas, int shares) {
  constexpr int RP = ExtendShape<D, NT>::RP;
  griddep_wait();
  const int c0 = static_cast<int>(blockIdx.x) / shares, share = static_cast<int>(blockIdx.x) - c0 * shares;
  const int4 s = __ldcg(reinterpret_cast<const int4*>(p.split) + 2 * c0);
  const int nf = s.x, b = s.y, kvh = s.z, row0 = s.w;
  if (nf < 2) return;
  const int rows = __ldcg(p.split + 8 * c0 + 4);
  const float4* part_o = reinterpret_cast<const float4*>(p.part);
  const float2* part_l = reinterpret_cast<const float2*>(p.part + 2LL * ctas * RP * D);
  auto slot_of = [&](int c) { return 2 * (c0 + min(c, nf - 1)) + (c == 0 ? 1 : 0); };
  for (int i = share * EXTEND_JOIN_THREADS + static_cast<int>(threadIdx.x); i < rows * (D / 8); i += shares * EXTEND_JOIN_THREADS) {
    const int c8 = small_div(i, rows), r = i - c8 * rows;
    float2 top = make_float2(-INFINITY, 0.f);
    float sum = 0.f, a[8] = {};
#pragma unroll 1
    for (int f0 = 0; f0 < nf; f0 += 4) {
      float2 ls[4];
      float4 o[4][2];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const long long slot = slot_of(f0 + f);
        ls[f] = __ldcg(part_l + slot * RP + r);
        o[f][0] = __ldcg(part_o + (slot * (D / 4) + 2 * c8) * RP + r);
        o[f][1] = __ldcg(part_o + (slot * (D / 4) + 2 * c8 + 1) * RP + r);
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        if (f0 + f >= nf || ls[f].x == -INFINITY) continue;  // (of the latter nothing was left but this)
        const float d = top.x == -INFINITY ? INFINITY : (ls[f].x - top.x) + (ls[f].y - top.y);
        const float e = ex2(-fabsf(d)), scale = d > 0.f ? e : 1.f, w = d > 0.f ? 1.f : e;  // (NaN where one is)
        if (d > 0.f) top = ls[f];
        const float v[8] = {o[f][0].x, o[f][0].y, o[f][0].z, o[f][0].w, o[f][1].x, o[f][1].y, o[f][1].z, o[f][1].w};
        sum = sum * scale + w;
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] = a[k] * scale + v[k] * w;
      }
    }
    const float inv = 1.0f / sum;
    const int ra = row0 + r, t = small_div(ra, p.G);
    const long long row = (static_cast<long long>(b) * p.Hq + kvh * p.G + (ra - t * p.G)) * p.T + t;
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = p.bf16 ? pack2<true>(a[2 * k] * inv, a[2 * k + 1] * inv) : pack2<false>(a[2 * k] * inv, a[2 * k + 1] * inv);
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (row * D + 8 * c8) * 2) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

}  // namespace du
