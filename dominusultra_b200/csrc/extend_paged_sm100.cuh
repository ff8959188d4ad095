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
// key scale, the softmax scale and the query row's own factor) the carried weight is 2^(x - m + 11) =
// w vs up to a row's constant, an fp16 value of at most 2^15 since m moves when some x exceeds it by 4,
// and the sum takes 2^(vr - log2 vs) times the sum of a group's weights, vr being the log2 of the first
// value scale of the fragment. Where a value scale is beyond 2^30 of that (then, and for the rest of the
// fragment) the sum has exponentials and a reference of its own: a key whose carried weight is nothing
// beside another's can have all of the softmax's. fp16 holds weights down to 2^-25 of a row's largest at
// full precision and to 2^-36 at all. Query rows are carried as fp16 with a power of two for each row.
//
// Work: the items' key tiles, item by item, cut into equal ranges, one per CTA of a persistent grid (an
// item's beginning is charged with PEN tiles). Lengths are read on the device; every CTA repeats the sum
// over them. An item within one CTA is written at once; the fragments of others leave fp32 partials, and
// the CTA that leaves the last one joins them.
//
// NT = 2 (more than 128 rows in an item, head_dim up to 128): two tiles of 128 rows, whose softmax
// warpgroups alternate with the tensor core. At head_dim 128 P overwrites S in tensor memory, and O_x += P_x V
// comes before the next S_x, so that S_x being there means that O_x is (products of the same shape
// complete in order); below that P has columns of its own, and the next S_x is computed as soon as S_x
// is read. NT = 1: one tile, two buffers of S, P over S. With CS = 4 (up to 32 rows) the rows stand in all four 32-lane parts of the tile, and each warp takes a quarter of
// a key tile's columns (P is zero in the others): the softmax of few rows is done by all four warps. Each
// part has a maximum, sum and O of its own, joined at the fragment's end.
//
// Warps (512 threads): 0-3 softmax (of the first row tile); 4-7 softmax of the second, or widening K;
// 8-11 widening (of both, or of V); 12 and 13 bulk copies of K and of V; 14 TMEM and MMA; 15 walks the
// fragments and fetches the scales. Every wait is bounded.
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
  int* cnt;           // tickets, zero between calls; the last one counts the CTAs that are done
  float* part;        // [2 gridDim.x][rows][D] partial outs, then [2 gridDim.x][rows] log2 of their sums, in two parts
  int done;           // index of the last ticket
  int max_len;        // tokens that the table's row and the rope tables cover
  int bf16;
  int B, Hq, Hkv, G, T, N, width;
  int block, block_log2;
  float scale_log2;
};

constexpr int EXTEND_THREADS = 512;
constexpr float EXTEND_TOP = 11.0f;   // log2 of the weight at a row's reference
constexpr float EXTEND_MOVE = 4.0f;   // how far beyond its reference a row's maximum may be
constexpr float EXTEND_LARGE = 1024.0f;  // references beyond this are kept in two parts
constexpr float EXTEND_FAR = 30.0f;   // how far a value scale may be from the fragment's first

template <int D_, int NT_, int CS_>
struct ExtendShape {
  static constexpr int D = D_, NT = NT_, CS = CS_;
  static constexpr int R = 128 / CS;             // rows of a tile
  static constexpr int RP = NT * R;              // rows of an item
  static constexpr int KT = D == 256 ? 64 : 128; // keys of a tile
  static constexpr int NC = KT / CS;             // columns of a key tile that a softmax thread takes
  static constexpr int SPAN = 2 * D >= 128 ? 128 : 2 * D;  // bytes per row of a swizzled block
  static constexpr int NBLK = 2 * D / SPAN;
  static constexpr int GPT = KT / 16;            // groups of 16 keys in a tile
  static constexpr int NB = 32 / GPT;            // tiles of a batch of scales
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int T_BYTES = KT * D * 2;     // a widened tile
  static constexpr int RAW = KT * D;             // a tile as it is cached
  static constexpr int NK = 2, NV = D == 256 ? 1 : 2;  // widened tiles
  static constexpr int MISC = CS > 1 ? 2560 : 2048;
  static constexpr int TILES = (231424 - MISC - NT * Q_BYTES - (NK + NV) * T_BYTES) / RAW;
  static constexpr int NRV = TILES / 2 > 8 ? 8 : TILES / 2;            // cached tiles of V in flight
  static constexpr int NRK = TILES - NRV > 8 ? 8 : TILES - NRV;        // and of K
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
  static constexpr int OFF_LSE = OFF_FRAG + NF * 64;   // [128] sums of the parts of a row, in two parts (CS > 1)
  static constexpr int OFF_BAR = OFF_LSE + (CS > 1 ? 1024 : 0);
  static constexpr int B_RKF = 0, B_RKE = B_RKF + NRK, B_RVF = B_RKE + NRK, B_RVE = B_RVF + NRV, B_KF = B_RVE + NRV,
                       B_KE = B_KF + NK, B_VF = B_KE + NK, B_VE = B_VF + NV, B_SCF = B_VE + NV, B_SCE = B_SCF + 2,
                       B_QF = B_SCE + 2, B_SF = B_QF + 2, B_SR = B_SF + 2, B_PF = B_SR + 2, B_OD = B_PF + 2, B_FF = B_OD + 2,
                       B_FE = B_FF + NF, B_GS = B_FE + NF, B_DR = B_GS + 1, N_BAR = B_DR + 1;
  static constexpr int OFF_WORDS = OFF_BAR + 8 * N_BAR;  // TMEM address, failed, flag
  static constexpr int SMEM_BYTES = OFF_WORDS + 16 + 1024;
  static constexpr int TM_S = 0;       // + x KT, x the row tile or the buffer
  static constexpr int TM_O = 2 * KT;  // + x D
  static constexpr bool SEP = NT == 2 && D < 128;            // P in columns of its own
  static constexpr int TM_P = SEP ? TM_O + NT * D : TM_S;    // + x KT / 2, or where S is
  static constexpr int TMEM_COLS = TM_O + NT * D + (SEP ? KT : 0) <= 256 ? 256 : 512;
  // Softmax warps, and the warps that widen K and V.
  static constexpr int SW = 4 * NT;
  static constexpr int CK = NT == 2 ? 2 : 4, CV = CK;
  static constexpr int REG_SOFTMAX = NT == 2 ? 192 : 216;
  static constexpr int REG_WIDEN = NT == 2 ? 80 : 104;
  static constexpr int REG_REST = NT == 2 ? 48 : 88;
  static constexpr int REGS = NT == 2 ? 2 * REG_SOFTMAX + REG_WIDEN + REG_REST : REG_SOFTMAX + 2 * REG_WIDEN + REG_REST;
  static constexpr int PEN = 3;
  static_assert(NT == 1 || (CS == 1 && 2 * KT + 2 * D <= 512), "two row tiles");
  static_assert(TM_O + NT * D + (SEP ? KT : 0) <= 512, "tensor memory");
  static_assert(NRV >= 1 && NRK >= 1 && NRK >= NRV, "cached tiles in flight");
  static_assert(OFF_WORDS + 16 - OFF_MISC <= MISC, "the small things' shared memory");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
  static_assert(OFF_FRAG % 16 == 0 && OFF_BAR % 8 == 0 && SC_BYTES % 16 == 0 && OFF_MISC % 16 == 0, "alignment");
  static_assert(REGS * 128 <= 65536, "register split");
};

// One fragment, as warp 15 leaves it for the other warps (16 words).
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
template <typename S>
struct ExtendWalk {
  long long cur, hi, base, per;  // base: position of the current item's beginning
  int b, kvh, item, past, len, items;
  // Key tiles of an item's rows up to `row` of (b, kvh).
  __device__ __forceinline__ static int tiles(const ExtendPagedParams& p, int past, int row) { return (past + row / p.G) / S::KT + 1; }
  __device__ __forceinline__ static int item_tiles(const ExtendPagedParams& p, int past, int n, int i) {
    return tiles(p, past, min(n * p.G, (i + 1) * S::RP) - 1);
  }
  __device__ __forceinline__ static int items_of(const ExtendPagedParams& p, int n) { return (n * p.G + S::RP - 1) / S::RP; }
  // Positions of one KV head of request b (a lane's own b).
  __device__ __forceinline__ static int span(const ExtendPagedParams& p, int b) {
    int past, len;
    const int n = extend_new(p, b, past, len);
    if (n <= 0) return 0;
    int sum = 0;
    const int k = items_of(p, n);
    for (int i = 0; i < k; ++i) sum += item_tiles(p, past, n, i) + S::PEN;
    return sum;
  }
  __device__ __forceinline__ void enter(const ExtendPagedParams& p) {
    const int n = extend_new(p, b, past, len);
    items = n > 0 ? items_of(p, n) : 0;
  }
  __device__ __forceinline__ void init(const ExtendPagedParams& p, int lane) {
    long long total = 0;
    for (int i = lane; i < p.B; i += 32) total += span(p, i);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= p.Hkv;
    const long long grid = gridDim.x;
    per = (total + grid - 1) / grid;
    cur = min(per * blockIdx.x, total);
    hi = min(cur + per, total);
    base = 0;
    b = kvh = item = items = 0;
    if (cur >= hi) return;
    // The request that holds `cur`.
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const long long own = b0 + lane < p.B ? static_cast<long long>(span(p, b0 + lane)) * p.Hkv : 0;
      long long in = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, cur < base + in);
      if (hit) {
        const int l = __ffs(static_cast<int>(hit)) - 1;
        b = b0 + l;
        base += __shfl_sync(0xffffffffu, in - own, l);
        const long long one = __shfl_sync(0xffffffffu, own, l) / p.Hkv;
        kvh = static_cast<int>((cur - base) / one);
        base += kvh * one;
        break;
      }
      base += __shfl_sync(0xffffffffu, in, 31);
    }
    enter(p);
    while (true) {
      const int cost = item_tiles(p, past, len - past, item) + S::PEN;
      if (cur < base + cost) break;
      base += cost;
      ++item;
    }
  }
  __device__ __forceinline__ bool next(const ExtendPagedParams& p, ExtendFrag& f) {
    while (true) {
      if (cur >= hi) return false;
      while (item >= items) {  // on to the next KV head, or the next request that has items
        item = 0;
        if (items == 0 || ++kvh == p.Hkv) {
          kvh = 0;
          ++b;
          enter(p);
        }
      }
      const int n = len - past;
      const int nk = item_tiles(p, past, n, item);
      const long long first = base + S::PEN, end = first + nk;
      const int j0 = static_cast<int>(max(cur - first, 0LL));
      const int j1 = static_cast<int>(min(hi, end) - first);
      cur = min(hi, end);
      if (j1 > 0) {
        f.kind = 1;
        f.b = b;
        f.kvh = kvh;
        f.row0 = item * S::RP;
        f.rows = min(n * p.G - f.row0, S::RP);
        f.past = past;
        f.len = len;
        f.j0 = j0;
        f.j1 = j1;
        f.nk0 = tiles(p, past, f.row0 + min(f.rows, S::R) - 1);
        f.nk1 = f.rows > S::R ? nk : 0;
        f.c0 = static_cast<int>(first / per);
        f.nf = static_cast<int>((end - 1) / per) - f.c0 + 1;
        f.slot = 2 * static_cast<int>(blockIdx.x) + (j0 > 0 ? 0 : 1);
      }
      if (cur == end) {
        base = end;
        ++item;
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

// One more part of a row's sum, y, beside those that `sum` counts relative to `top` (logarithms in two
// parts; -inf: nothing); `share` is the caller's own part relative to `top`, y if `mine`.
__device__ __forceinline__ void join_sums(float2& top, float& sum, float& share, float2 y, bool mine) {
  if (y.x == -INFINITY) return;
  float scale = 1.f, w = 1.f;
  if (top.x == -INFINITY) {
    top = y;
  } else {
    const float d = (y.x - top.x) + (y.y - top.y);
    if (d > 0.f) {
      scale = exp2f(-d);
      top = y;
    } else {
      w = exp2f(d);  // (NaN where one is)
    }
  }
  sum = sum * scale + w;
  share = mine ? w : share * scale;
}

template <int D, int NT, int CS>
__global__ void __launch_bounds__(EXTEND_THREADS, 1) extend_paged_kernel(const ExtendPagedParams p) {
  using S = ExtendShape<D, NT, CS>;
  constexpr int KT = S::KT, NC = S::NC, R = S::R, RP = S::RP, SPAN = S::SPAN, GPT = S::GPT, NB = S::NB;
  constexpr int NK = S::NK, NV = S::NV, NRK = S::NRK, NRV = S::NRV, NF = S::NF;
  constexpr uint32_t SWZ = swizzle_code(SPAN);
  constexpr uint32_t IDESC_QK = idesc_f16(128, KT, 0, 0, 0, 0);
  constexpr uint32_t IDESC_PV = idesc_f16(128, D, 0, 0, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t sbase = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw_u32);
  auto bar = [&](int i) -> uint32_t { return sbase + S::OFF_BAR + 8u * static_cast<uint32_t>(i); };
  auto RKF = [&](int s) { return bar(S::B_RKF + s); };  // cached tile of K landed
  auto RKE = [&](int s) { return bar(S::B_RKE + s); };  // and widened
  auto RVF = [&](int s) { return bar(S::B_RVF + s); };
  auto RVE = [&](int s) { return bar(S::B_RVE + s); };
  auto KF = [&](int s) { return bar(S::B_KF + s); };    // widened K written
  auto KE = [&](int s) { return bar(S::B_KE + s); };    // and multiplied
  auto VF = [&](int s) { return bar(S::B_VF + s); };
  auto VE = [&](int s) { return bar(S::B_VE + s); };
  auto SCF = [&](int s) { return bar(S::B_SCF + s); };  // batch of scales written
  auto SCE = [&](int s) { return bar(S::B_SCE + s); };  // read by the softmax warps and those that widen V
  auto QF = [&](int x) { return bar(S::B_QF + x); };    // query rows written
  auto SF = [&](int x) { return bar(S::B_SF + x); };    // S (of row tile x, or in buffer x) complete
  auto SR = [&](int x) { return bar(S::B_SR + x); };    // S_x read (SEP)
  auto PF = [&](int x) { return bar(S::B_PF + x); };    // P written
  auto OD = [&](int x) { return bar(S::B_OD + x); };    // P V of a tile done; with P over two S: O_x final
  auto FF = [&](int i) { return bar(S::B_FF + i); };    // fragment entry written
  auto FE = [&](int i) { return bar(S::B_FE + i); };    // and read by every warp but the walker
  const uint32_t BAR_GS = bar(S::B_GS);                 // the softmax warps among themselves
  const uint32_t BAR_DR = bar(S::B_DR);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(sgen + S::OFF_WORDS);
  volatile int* failed = reinterpret_cast<volatile int*>(sgen + S::OFF_WORDS + 4);
  volatile int* joins = reinterpret_cast<volatile int*>(sgen + S::OFF_WORDS + 8);
  volatile int* frags = reinterpret_cast<volatile int*>(sgen + S::OFF_FRAG);

  if (tid == 0) {
    for (int s = 0; s < NRK; ++s) {
      mbar_init(RKF(s), 1);
      mbar_init(RKE(s), S::CK);
    }
    for (int s = 0; s < NRV; ++s) {
      mbar_init(RVF(s), 1);
      mbar_init(RVE(s), S::CV);
    }
    for (int s = 0; s < NK; ++s) {
      mbar_init(KF(s), S::CK);
      mbar_init(KE(s), 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(VF(s), S::CV);
      mbar_init(VE(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(SCF(s), 1);
      mbar_init(SCE(s), S::SW + S::CV);
      mbar_init(QF(s), 4);
      mbar_init(SF(s), 1);
      mbar_init(SR(s), 4);
      mbar_init(PF(s), 4);
      mbar_init(OD(s), 1);
    }
    for (int s = 0; s < NF; ++s) {
      mbar_init(FF(s), 1);
      mbar_init(FE(s), 15);
    }
    mbar_init(BAR_GS, S::SW);
    mbar_init(BAR_DR, 1);
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

  // The next fragment, for every warp but the walker; kind 0: none (or a wait expired).
  int n_frag = 0;
  auto take = [&]() -> ExtendFrag {
    ExtendFrag f;
    const int s = n_frag % NF;
    bool ok = mbar_wait(FF(s), (n_frag / NF) & 1, failed, 500);
    ok = __all_sync(0xffffffffu, ok);
    const volatile int* e = frags + 16 * s;
    f.kind = ok ? e[0] : 0;
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

  if (warp < S::SW) {
    // ------------------------------------------------------------------ softmax
    regs_inc<S::REG_SOFTMAX>();
    const int x = warp >> 2, w4 = warp & 3;
    const int lane128 = 32 * w4 + lane;   // TMEM lane
    const int row = lane128 % R;          // row of the tile
    const int col0 = (lane128 / R) * NC;  // first column of a key tile that this thread takes
    const uint32_t lane_off = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t q_tile = sbase + S::OFF_Q + x * S::Q_BYTES;
    const int stid = tid;                 // thread among the softmax warps
    constexpr int ST = 32 * S::SW;
    int n_tile = 0, n_batch = 0, n_of = 0, n_gs = 0;
    auto group_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR_GS);
      const bool w = mbar_wait(BAR_GS, n_gs++ & 1, failed, 501);
      return __all_sync(0xffffffffu, w);
    };
    bool ok = true;
    while (ok) {
      const ExtendFrag f = take();
      if (f.kind == 0) break;
      const int nt = f.j1 - f.j0;                                     // key tiles of the fragment
      const int n = max(0, min(f.j1, x ? f.nk1 : f.nk0) - f.j0);      // and of this row tile
      const int r_item = x * R + row;                                 // row of the item
      const bool row_ok = r_item < f.rows;
      const int r_all = f.row0 + min(r_item, f.rows - 1);
      const int t = r_all / p.G;                                      // its token and head
      const int h = f.kvh * p.G + (r_all - t * p.G);
      const long long q_row = (static_cast<long long>(f.b) * p.Hq + h) * p.T + t;
      const int kmax = f.past + t;                                    // the last key that it sees
      const int kmin = f.past + (f.row0 + x * R) / p.G;               // that every row of the tile sees
      float qs = 0.f;  // the row's factor
      if (n > 0) {
        // The query row: rotated in fp32, times a power of two that brings its largest input to
        // [2^8, 2^9), as fp16.
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + q_row * (2 * D);
        const uint8_t* cp = static_cast<const uint8_t*>(p.cos) + static_cast<long long>(kmax) * D;
        const uint8_t* sp = static_cast<const uint8_t*>(p.sin) + static_cast<long long>(kmax) * D;
        uint4 v[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) v[i] = ldg_v4(src + 16 * i);
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = __vmaxu2(top, u[k] & 0x7fff7fffu);
        }
        const float2 tops = p.bf16 ? split2<true>(top) : split2<false>(top);
        const uint32_t top_bits = __float_as_uint(fmaxf(tops.x, tops.y));
        int e = static_cast<int>(top_bits >> 23) - 127;
        if (e == -127 || e == 128) e = 8;  // (zero, or not finite)
        e = min(max(e - 8, -100), 100);
        const float up = __int_as_float((127 - e) << 23);
        qs = __int_as_float((127 + e) << 23);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint4 c = ldg_v4(cp + 16 * i), s = ldg_v4(sp + 16 * i);
          const uint4 a = v[i], b = v[i + D / 16];
          const uint32_t ca[4] = {c.x, c.y, c.z, c.w}, sa[4] = {s.x, s.y, s.z, s.w};
          const uint32_t aa[4] = {a.x, a.y, a.z, a.w}, ba[4] = {b.x, b.y, b.z, b.w};
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 fc = p.bf16 ? split2<true>(ca[k]) : split2<false>(ca[k]);
            const float2 fs = p.bf16 ? split2<true>(sa[k]) : split2<false>(sa[k]);
            float2 fa = p.bf16 ? split2<true>(aa[k]) : split2<false>(aa[k]);
            float2 fb = p.bf16 ? split2<true>(ba[k]) : split2<false>(ba[k]);
            fa.x *= up;
            fa.y *= up;
            fb.x *= up;
            fb.y *= up;
            lo[k] = pack2<false>(fa.x * fc.x - fb.x * fs.x, fa.y * fc.y - fb.y * fs.y);
            hi[k] = pack2<false>(fb.x * fc.x + fa.x * fs.x, fb.y * fc.y + fa.y * fs.y);
          }
          st_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, lane128, i), make_uint4(lo[0], lo[1], lo[2], lo[3]));
          st_shared_v4(q_tile + swz_chunk_offset<SPAN>(128, lane128, i + D / 16), make_uint4(hi[0], hi[1], hi[2], hi[3]));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(QF(x));
      }
      const uint32_t o_addr = tmem + lane_off + S::TM_O + x * D;
      // The reference of the weights is m + mlo (log2 domain); mlo is 0 but for references so large that
      // a sum with log2 vs would round away. l: the sum of 2^(s + vr - m - mlo + 11), with `far` of
      // 2^(s - m - eo).
      float m = -INFINITY, mlo = 0.f, l = 0.f, eo = -INFINITY, vr = 0.f;
      bool far = false;
      for (int jj = 0; ok && jj < nt; ++jj) {
        const int bs = n_batch & 1;
        const uint8_t* sc = sgen + S::OFF_SC + bs * S::SC_BYTES;
        if (jj % NB == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(SCF(bs), (n_batch >> 1) & 1, failed, 502));
          if (!ok) break;
          const bool now = *reinterpret_cast<const int*>(sc + 384 + 4 * NB + 4) != 0;
          if (jj == 0) vr = *reinterpret_cast<const float*>(sc + 384 + 4 * NB);
          if (now && !far) {
            far = true;
            eo = l == 0.f ? -INFINITY : mlo - EXTEND_TOP - vr;
          }
        }
        if (jj < n) {
          const int sb = NT == 2 ? x : n_tile & 1;
          const uint32_t s_addr = tmem + lane_off + S::TM_S + sb * KT;
          const uint32_t p_addr = S::SEP ? tmem + lane_off + S::TM_P + x * (KT / 2) : s_addr;
          ok = mbar_wait(SF(sb), (NT == 2 ? n_tile : n_tile >> 1) & 1, failed, 503);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          float s[NC];
          const int k0 = (f.j0 + jj) * KT + col0;
          const bool diag = (f.j0 + jj) * KT + KT - 1 > kmin;  // some key of the tile is hidden from some row
#pragma unroll
          for (int c = 0; c < NC; c += 16) tmem_ld16(s_addr + col0 + c, s + c);
          float kq[NC / 16], lv[NC / 16];
          const int g0 = (jj % NB) * GPT + col0 / 16;
#pragma unroll
          for (int g = 0; g < NC / 16; ++g) {
            kq[g] = reinterpret_cast<const float*>(sc)[g0 + g] * qs;
            lv[g] = reinterpret_cast<const float*>(sc + 128)[g0 + g];
          }
          tmem_wait_ld();
          if (diag) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
              if (k0 + c > kmax) s[c] = -INFINITY;
          }
          if constexpr (S::SEP) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(SR(x));  // S is in registers: the next one may overwrite it
          }
          float mx = -INFINITY, ga[NC / 16];
#pragma unroll
          for (int g = 0; g < NC / 16; ++g) {
            float a = fmaxf(s[16 * g], s[16 * g + 1]), b = fmaxf(s[16 * g + 2], s[16 * g + 3]);
#pragma unroll
            for (int c = 4; c < 16; c += 4) {
              a = max3(a, s[16 * g + c], s[16 * g + c + 1]);
              b = max3(b, s[16 * g + c + 2], s[16 * g + c + 3]);
            }
            ga[g] = fmaxf(a, b);
            mx = fmaxf(mx, fmaf(ga[g], kq[g], lv[g]));
          }
          const float m_old = m, mlo_old = mlo;
          bool moved = mx > m + mlo + EXTEND_MOVE;
          float base = 0.f;  // what is subtracted from log2 vs
          const bool large = (fabsf(m) > EXTEND_LARGE && m != -INFINITY) || (fabsf(mx) > EXTEND_LARGE && mx != -INFINITY);
          if (!far && !__any_sync(0xffffffffu, large)) {
            if (moved) {
              m = mx;
              mlo = 0.f;
            }
            if (m != -INFINITY) base = m + mlo;
          } else {
            // Scores relative to the reference first, then the rest: nothing is rounded away beside a
            // large score. The product is rounded before the difference is taken, so that scores that are
            // alike have the same weight whatever their size.
            auto less = [](float a, float k, float r) { return __fadd_rn(__fmul_rn(a, k), -r); };
            float hi = -INFINITY, lo = -INFINITY;
#pragma unroll
            for (int g = 0; g < NC / 16; ++g) hi = fmaxf(hi, ga[g] * kq[g]);
            const float h0 = hi == -INFINITY ? 0.f : hi;
#pragma unroll
            for (int g = 0; g < NC / 16; ++g) lo = fmaxf(lo, less(ga[g], kq[g], h0) + lv[g]);
            moved = m == -INFINITY ? hi != -INFINITY : (hi - m) + (lo - mlo) > EXTEND_MOVE;
            if (moved) {
              m = hi;
              mlo = lo;
            }
            const float mr = m == -INFINITY ? 0.f : m;
            base = m == -INFINITY ? 0.f : mlo;
            float es = -INFINITY;
#pragma unroll
            for (int g = 0; g < NC / 16; ++g) es = fmaxf(es, less(ga[g], kq[g], mr));
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c] = less(s[c], kq[c / 16], mr);
#pragma unroll
            for (int g = 0; g < NC / 16; ++g) kq[g] = 1.f;
            if (far) {
              // value scales far apart: the sum has a reference of its own
              if (moved && m_old != -INFINITY) eo += m_old - m;
              const float en = fmaxf(l == 0.f ? -INFINITY : eo, es), e0 = en == -INFINITY ? 0.f : en;
              l = l == 0.f ? 0.f : l * exp2f(eo - e0);
              eo = en;
#pragma unroll
              for (int c = 0; c < NC; ++c) {
                const float w = exp2f(s[c] - e0);
                if (!diag || k0 + c <= kmax) l += w;
              }
            }
          }
          uint64_t acc = f2(0.f, 0.f);
          uint32_t pk[NC / 2];
#pragma unroll
          for (int g = 0; g < NC / 16; ++g) {
            const float add = lv[g] - base + EXTEND_TOP;
            const uint64_t A = f2(add, add), K = f2(kq[g], kq[g]);
            uint64_t sum = f2(0.f, 0.f);
#pragma unroll
            for (int c = 16 * g; c < 16 * g + 16; c += 2) {
              const float2 xx = f2_split(f2_fma(f2(s[c], s[c + 1]), K, A));
              float2 pp = make_float2(ex2(xx.x), ex2(xx.y));
              if (diag) {
                if (k0 + c > kmax) pp.x = 0.f;
                if (k0 + c + 1 > kmax) pp.y = 0.f;
              }
              sum = f2_add(sum, f2(pp.x, pp.y));
              pk[c / 2] = pack2<false>(pp.x, pp.y);
            }
            const float iv = reinterpret_cast<const float*>(sc + 256)[g0 + g];
            acc = f2_fma(sum, f2(iv, iv), acc);
          }
          if ((NT == 1 || S::SEP) && jj > 0) {
            // The product before must be done with O, and with P where that is not over S. (Waited for in
            // every tile: a parity tells only two phases apart.)
            ok = __all_sync(0xffffffffu, mbar_wait(OD(x), (n_tile - 1) & 1, failed, 504));
            if (!ok) break;
            tc_fence_after();
          }
          if (jj > 0 && __any_sync(0xffffffffu, moved)) {
            const float alpha = moved && m_old != -INFINITY ? ex2((m_old - m) + (mlo_old - mlo)) : 1.0f;
            if (!far) l *= alpha;
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(o_addr + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16(o_addr + c, o);
            }
          }
          if (!far) {
            const float2 rs = f2_split(acc);
            l += rs.x + rs.y;
          }
          if constexpr (CS == 1) {
#pragma unroll
            for (int c = 0; c < NC / 2; c += 16) tmem_st16u(p_addr + c, pk + c);
          } else {
            // this thread's columns of P, zeros in the others
            uint32_t z[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = 0u;
            if constexpr (NC >= 32) {
#pragma unroll
              for (int c = 0; c < KT / 2; c += 16) {
                const int mine = c - col0 / 2;
                if (mine >= 0 && mine < NC / 2) {
                  if constexpr (NC == 32) tmem_st16u(p_addr + c, pk);
                  else if (mine == 0) tmem_st16u(p_addr + c, pk);
                  else tmem_st16u(p_addr + c, pk + 16);
                } else {
                  tmem_st16u(p_addr + c, z);
                }
              }
            } else {  // (NC = 16: eight columns)
#pragma unroll
              for (int c = 0; c < KT / 2; c += 16) {
                uint32_t y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = (c + i) / 8 == col0 / 16 ? pk[i % 8] : 0u;
                tmem_st16u(p_addr + c, y);
              }
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(PF(sb));
          ++n_tile;
        }
        if (jj % NB == NB - 1 || jj == nt - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(SCE(bs));
          ++n_batch;
        }
      }
      if (!ok) break;
      if (n > 0) {
        ok = mbar_wait(OD(x), (NT == 2 && !S::SEP ? n_of++ : n_tile - 1) & 1, failed, 505);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
      }
      // The log2 of the row's (or its part's) sum, in two parts; and what brings O to the fragment's output,
      // O 2^(m + mlo - 11) over the sum, in two factors since the exponent may be large.
      const float2 lse = l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m, lg2(l) + (far ? eo : mlo - EXTEND_TOP - vr));
      float w1 = 0.f, w2 = 0.f;
      if (l != 0.f) {
        const float ex = far ? mlo - EXTEND_TOP - eo : vr, half = rintf(0.5f * ex);
        w2 = exp2f(half);
        w1 = exp2f(ex - half) / l;
      }
      float* part_o = p.part;
      float2* part_l = reinterpret_cast<float2*>(p.part + 2LL * gridDim.x * RP * D);
      if constexpr (CS == 1) {
        if (f.nf > 1 && row_ok) part_l[static_cast<long long>(f.slot) * RP + r_item] = lse;
        if (n > 0) {
          float* dst = part_o + (static_cast<long long>(f.slot) * RP + r_item) * D;
          uint8_t* out = static_cast<uint8_t*>(p.out) + q_row * (2 * D);
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_ld16(o_addr + c, o);
            tmem_wait_ld();
            if (row_ok) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = o[i] * w1 * w2;
              if (f.nf > 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(dst + c)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              } else {
                uint32_t u[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = p.bf16 ? pack2<true>(o[2 * i], o[2 * i + 1]) : pack2<false>(o[2 * i], o[2 * i + 1]);
                reinterpret_cast<uint4*>(out + 2 * c)[0] = make_uint4(u[0], u[1], u[2], u[3]);
                reinterpret_cast<uint4*>(out + 2 * c)[1] = make_uint4(u[4], u[5], u[6], u[7]);
              }
            }
          }
        }
      } else {
        // The parts of a row joined: their weights by their sums, O half the columns at a time where
        // the query rows were (a row's 16-byte pieces turned by the row's number).
        float2* lses = reinterpret_cast<float2*>(sgen + S::OFF_LSE);
        lses[lane128] = lse;
        if (!(ok = group_sync())) break;
        float2 top = lses[row];
        float sum = 1.f, share = lane128 < R ? 1.f : 0.f;  // relative to `top`
        if (top.x == -INFINITY) sum = share = 0.f;
#pragma unroll
        for (int c = 1; c < CS; ++c) {
          const float2 y = lses[c * R + row];
          join_sums(top, sum, share, y, lane128 / R == c);
        }
        w1 *= share / sum;
        if (sum == 0.f) w1 = 0.f;
        if (sum != sum) w1 = sum;  // (a part that is not a number)
        if (f.nf > 1 && lane128 < R && row_ok)
          part_l[static_cast<long long>(f.slot) * RP + row] = sum == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(top.x, top.y + lg2(sum));
        constexpr int PC = D / 8;  // 16-byte pieces of half a row
        float4* buf = reinterpret_cast<float4*>(sgen + S::OFF_Q);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int c = 0; c < D / 2; c += 8) {
            float o[8];
            uint32_t u[8];
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                         : "r"(o_addr + half * (D / 2) + c)
                         : "memory");
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(u[i]) * w1 * w2;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              buf[lane128 * PC + (c / 4 + i + lane128) % PC] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          if (!(ok = group_sync())) break;
          for (int i = stid; i < min(f.rows, R) * PC; i += ST) {
            const int rr = i / PC, k = i - rr * PC;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < CS; ++c) {
              const float4 o = buf[(c * R + rr) * PC + (k + c * R + rr) % PC];
              a.x += o.x;
              a.y += o.y;
              a.z += o.z;
              a.w += o.w;
            }
            const int col = half * (D / 2) + 4 * k;
            if (f.nf > 1) {
              *reinterpret_cast<float4*>(part_o + (static_cast<long long>(f.slot) * RP + rr) * D + col) = a;
            } else {
              const int ra = f.row0 + rr, tt = ra / p.G;
              const long long orow = (static_cast<long long>(f.b) * p.Hq + f.kvh * p.G + (ra - tt * p.G)) * p.T + tt;
              uint2 u;
              u.x = p.bf16 ? pack2<true>(a.x, a.y) : pack2<false>(a.x, a.y);
              u.y = p.bf16 ? pack2<true>(a.z, a.w) : pack2<false>(a.z, a.w);
              *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + (orow * D + col) * 2) = u;
            }
          }
          if (!(ok = group_sync())) break;
        }
        if (!ok) break;
      }
      if (f.nf > 1) {
        // The last of the item's fragments joins them.
        if (!(ok = group_sync())) break;
        if (stid == 0) *joins = atom_add_acq_rel_gpu(p.cnt + f.c0, 1) == f.nf - 1;
        if (!(ok = group_sync())) break;
        if (*joins) {
          for (int i = stid; i < f.rows * (D / 4); i += ST) {
            const int rr = i / (D / 4), col = 4 * (i - rr * (D / 4));
            float2 top = make_float2(-INFINITY, 0.f);
            float sum = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < f.nf; ++c) {
              const int slot = 2 * (f.c0 + c) + (c == 0 ? 1 : 0);
              const float2 ls = __ldcg(part_l + static_cast<long long>(slot) * RP + rr);
              const float4 o = __ldcg(reinterpret_cast<const float4*>(part_o + (static_cast<long long>(slot) * RP + rr) * D + col));
              if (ls.x == -INFINITY) continue;
              float scale = 1.f, w = 1.f;
              if (top.x == -INFINITY) {
                top = ls;
              } else {
                const float d = (ls.x - top.x) + (ls.y - top.y);
                if (d > 0.f) {
                  scale = exp2f(-d);
                  top = ls;
                } else {
                  w = exp2f(d);
                }
              }
              a.x = a.x * scale + o.x * w;
              a.y = a.y * scale + o.y * w;
              a.z = a.z * scale + o.z * w;
              a.w = a.w * scale + o.w * w;
              sum = sum * scale + w;
            }
            const float inv = 1.0f / sum;
            const int ra = f.row0 + rr, tt = ra / p.G;
            const long long orow = (static_cast<long long>(f.b) * p.Hq + f.kvh * p.G + (ra - tt * p.G)) * p.T + tt;
            uint2 u;
            u.x = p.bf16 ? pack2<true>(a.x * inv, a.y * inv) : pack2<false>(a.x * inv, a.y * inv);
            u.y = p.bf16 ? pack2<true>(a.z * inv, a.w * inv) : pack2<false>(a.z * inv, a.w * inv);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + (orow * D + col) * 2) = u;
          }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ rows behind the last token
    regs_dec<S::REG_WIDEN>();
    {
      const int first = warp - S::SW, warps = 12 - S::SW;
      const int G16 = D / 8;  // 16-byte pieces of a row
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
          const long long s0 = static_cast<long long>(b) * p.Hq;
          const long long skip = (blockIdx.x + gridDim.x - s0 % gridDim.x) % gridDim.x;
          for (long long h = skip; h < p.Hq; h += gridDim.x) {
            uint4* dst = reinterpret_cast<uint4*>(p.out) + ((s0 + h) * p.T + from) * G16;
            const long long pieces = static_cast<long long>(p.T - from) * G16;
            for (long long i = 32 * first + lane; i < pieces; i += 32 * warps) dst[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
    }
    // ------------------------------------------------------------------ widening
    const bool values = NT == 2 ? warp >= 10 : warp >= 8;
    const int wt = (NT == 2 ? (warp & 1) : (warp & 3)) * 32 + lane;  // thread of this cache's warps
    constexpr int WT = 32 * S::CK;
    constexpr int CPR = D / 16;        // 16-byte pieces of a cached row
    constexpr int PIECES = KT * CPR;
    constexpr int PER = PIECES / WT;   // of a thread
    const int n_raw = values ? NRV : NRK, n_wide = values ? NV : NK;
    const int off_raw = values ? S::OFF_RV : S::OFF_RK, off_wide = values ? S::OFF_V : S::OFF_K;
    auto raw_full = [&](int s) { return values ? RVF(s) : RKF(s); };
    auto raw_empty = [&](int s) { return values ? RVE(s) : RKE(s); };
    auto wide_full = [&](int s) { return values ? VF(s) : KF(s); };
    auto wide_empty = [&](int s) { return values ? VE(s) : KE(s); };
    int rs = 0, rp = 0, ws = 0, wp = 1, n_batch = 0;  // stages and parities
    bool ok = true;
    while (ok) {
      const ExtendFrag f = take();
      if (f.kind == 0) break;
      const int nt = f.j1 - f.j0;
      for (int jj = 0; jj < nt; ++jj) {
        uint32_t zero = 0u;   // groups of V that are not to be used
        int rows_left = KT;   // rows up to the request's end
        if (values) {
          const int bs = n_batch & 1;
          if (jj % NB == 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(SCF(bs), (n_batch >> 1) & 1, failed, 510));
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
        ok = mbar_wait(raw_full(rs), rp, failed, 511) && mbar_wait(wide_empty(ws), wp, failed, 512);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t src = sbase + off_raw + rs * S::RAW, dst = sbase + off_wide + ws * S::T_BYTES;
        const bool clear = zero != 0u || (values && rows_left < KT);
#pragma unroll 4
        for (int i = 0; i < PER; ++i) {
          const int c = wt + i * WT, r = c / CPR, k = c % CPR;
          const uint4 b = ld_shared_v4(src + 16 * c);
          uint4 lo, hi;
          widen16(b, lo, hi);
          if (clear && (r >= rows_left || ((zero >> (r / 16)) & 1u))) lo = hi = make_uint4(0u, 0u, 0u, 0u);
          // (lanes of a quarter-warp that would meet in a bank write their halves in the other order)
          const bool turn = CPR >= 8 && (k & 4);
          st_shared_v4(dst + swz_chunk_offset<SPAN>(KT, r, 2 * k + turn), turn ? hi : lo);
          st_shared_v4(dst + swz_chunk_offset<SPAN>(KT, r, 2 * k + !turn), turn ? lo : hi);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(raw_empty(rs));
          mbar_arrive(wide_full(ws));
        }
        if (++rs == n_raw) {
          rs = 0;
          rp ^= 1;
        }
        if (++ws == n_wide) {
          ws = 0;
          wp ^= 1;
        }
      }
    }
  } else {
    regs_dec<S::REG_REST>();
    if (warp == 12 || warp == 13) {
      // ------------------------------------------------------------------ copies of K or V
      const bool values = warp == 13;
      const uint8_t* cache = values ? p.v8 : p.k8;
      const int n_raw = values ? NRV : NRK, off_raw = values ? S::OFF_RV : S::OFF_RK;
      auto full = [&](int s) { return values ? RVF(s) : RKF(s); };
      auto empty = [&](int s) { return values ? RVE(s) : RKE(s); };
      const int piece = min(p.block, KT);          // keys of a copy
      const uint32_t bytes = static_cast<uint32_t>(piece) * D;
      int st = 0, ph = 1;
      long long issued = 0;
      bool ok = true;
      while (ok) {
        const ExtendFrag f = take();
        if (f.kind == 0) break;
        const int nt = f.j1 - f.j0;
        const int* row = p.table + static_cast<long long>(f.b) * p.width;
        // A lane has a group of 16 keys of NB tiles; the ids of the next ones are fetched ahead.
        auto fetch = [&](int t0) {
          const int key = (f.j0 + t0) * KT + 16 * lane;
          return key < f.len ? row[key >> p.block_log2] : -1;
        };
        int id = fetch(0);
        for (int t0 = 0; ok && t0 < nt; t0 += NB) {
          const int next = t0 + NB < nt ? fetch(t0 + NB) : -1;
          const bool first = (16 * lane) % piece == 0 && static_cast<unsigned>(id) < static_cast<unsigned>(p.N);
          const int key = (f.j0 + t0) * KT + 16 * lane;
          const uint8_t* src = cache + ((static_cast<long long>(id) * p.Hkv + f.kvh) * p.block + (key & (p.block - 1))) * D;
          const unsigned firsts = __ballot_sync(0xffffffffu, first);
          for (int i = 0; i < NB && t0 + i < nt; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait(empty(st), ph, failed, 520));
            if (!ok) break;
            const unsigned mine = firsts & (((GPT == 32 ? 0u : (1u << GPT)) - 1u) << (i * GPT));
            if (lane == 0) mbar_expect_tx(full(st), __popc(mine) * bytes);
            __syncwarp();
            if ((mine >> lane) & 1u) bulk_load(sbase + off_raw + st * S::RAW + (lane % GPT) * 16 * D, src, bytes, full(st));
            ++issued;
            if (++st == n_raw) {
              st = 0;
              ph ^= 1;
            }
          }
          id = next;
        }
      }
      // Every copy lands before the CTA ends.
      for (long long i = issued > n_raw ? issued - n_raw : 0; i < issued; ++i)
        mbar_wait_drain(full(static_cast<int>(i % n_raw)), static_cast<uint32_t>((i / n_raw) & 1), 521);
    } else if (warp == 14) {
      // ------------------------------------------------------------------ MMA issuer
      const uint64_t dq0 = smem_desc(sbase + S::OFF_Q, 16, 8 * SPAN, SWZ);
      const uint64_t dk0 = smem_desc(sbase + S::OFF_K, 16, 8 * SPAN, SWZ);
      const uint64_t dv0 = smem_desc(sbase + S::OFF_V, KT * SPAN, 8 * SPAN, SWZ);
      const bool leader = elect_one();
      int ks = 0, kp = 0, vs = 0, vp = 0;      // stages and parities of widened K and V
      int n_q[2] = {0, 0}, n_s[2] = {0, 0}, n_p[2] = {0, 0};  // fragments, S and P tiles per row tile
      bool ok = true;
      auto wait = [&](uint32_t b, int parity, unsigned site) {
        return __all_sync(0xffffffffu, mbar_wait(b, parity, failed, site)) != 0;
      };
      while (ok) {
        const ExtendFrag f = take();
        if (f.kind == 0) break;
        const int nt = f.j1 - f.j0;
        int n[2] = {max(0, min(f.j1, f.nk0) - f.j0), NT == 2 ? max(0, min(f.j1, f.nk1) - f.j0) : 0};
        for (int x = 0; x < NT && ok; ++x)
          if (n[x] > 0) ok = wait(QF(x), n_q[x]++ & 1, 530);
        if (!ok) break;
        auto qk = [&](int x, int jj) {  // S of key tile jj (its widened K is there)
          if (jj >= n[x]) return;
          const int sb = NT == 2 ? x : n_s[0] & 1;
          // S may be written over: P there is multiplied (NT = 1; the shapes differ, so the order of the
          // products alone does not say so), or S is read
          if (NT == 1 && jj >= 2) ok = wait(OD(0), n_s[0] & 1, 535);  // (before: known from the query rows)
          if (S::SEP && n_s[x] >= 1) ok = wait(SR(x), (n_s[x] - 1) & 1, 536);
          if (!ok) return;
          tc_fence_after();
          if (leader) {
            const uint64_t dq = dq0 + static_cast<uint64_t>((x * S::Q_BYTES) >> 4);
            const uint64_t dk = dk0 + static_cast<uint64_t>((ks * S::T_BYTES) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off_q = ((kk * 32) / SPAN) * 128 * SPAN + (kk * 32) % SPAN;
              const uint32_t off_k = ((kk * 32) / SPAN) * KT * SPAN + (kk * 32) % SPAN;
              umma_f16_ss(tmem + S::TM_S + sb * KT, dq + (off_q >> 4), dk + (off_k >> 4), IDESC_QK, kk > 0 ? 1u : 0u);
            }
            umma_commit(SF(sb));
          }
          __syncwarp();
          ++n_s[x];
        };
        bool v_there = false;
        auto pv = [&](int x, int jj) -> bool {  // O of key tile jj
          if (jj < 0 || jj >= n[x]) return true;
          const int sb = NT == 2 ? x : n_p[0] & 1;
          if (!wait(PF(sb), (NT == 2 ? n_p[x] : n_p[0] >> 1) & 1, 531)) return false;
          if (!v_there && !wait(VF(vs), vp, 532)) return false;
          v_there = true;
          tc_fence_after();
          if (leader) {
            const uint64_t dv = dv0 + static_cast<uint64_t>((vs * S::T_BYTES) >> 4);
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk)
              umma_f16_ts(tmem + S::TM_O + x * D, tmem + (S::SEP ? S::TM_P + x * (KT / 2) : S::TM_S + sb * KT) + kk * 8,
                          dv + static_cast<uint64_t>((kk * 16 * SPAN) >> 4), IDESC_PV, (jj > 0 || kk > 0) ? 1u : 0u);
            if (NT == 1 || S::SEP || jj == n[x] - 1) umma_commit(OD(x));
          }
          __syncwarp();
          ++n_p[x];
          return true;
        };
        for (int jj = 0; ok && jj <= nt; ++jj) {
          const bool has_k = jj < nt;
          if (has_k && !(ok = wait(KF(ks), kp, 533))) break;
          v_there = false;
          if constexpr (NT == 1) {
            if (has_k) {
              qk(0, jj);
              if (leader) umma_commit(KE(ks));  // (before P V: the next K may be widened meanwhile)
            }
            ok = ok && pv(0, jj - 1);
          } else if constexpr (S::SEP) {
            if (has_k) {
              qk(0, jj);
              if (ok) qk(1, jj);
            }
            ok = ok && pv(0, jj - 1) && pv(1, jj - 1);
          } else {
            ok = pv(0, jj - 1);
            if (ok && has_k) qk(0, jj);
            ok = ok && pv(1, jj - 1);
            if (ok && has_k) qk(1, jj);
          }
          if (!ok) break;
          if (has_k) {
            if (NT == 2 && leader) umma_commit(KE(ks));
            if (++ks == NK) {
              ks = 0;
              kp ^= 1;
            }
          }
          if (jj > 0) {
            if (leader) umma_commit(VE(vs));
            if (++vs == NV) {
              vs = 0;
              vp ^= 1;
            }
          }
          __syncwarp();
        }
      }
      if (leader) {
        umma_commit(BAR_DR);
        mbar_wait_drain(BAR_DR, 0, 534);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------------ fragments and scales
      ExtendWalk<S> walk;
      walk.init(p, lane);
      int nfr = 0, n_batch = 0;
      bool ok = true;
      while (true) {
        ExtendFrag f{};
        const bool more = walk.next(p, f);
        if (!more) f.kind = 0;
        const int slot = nfr % NF;
        if (nfr >= NF) ok = __all_sync(0xffffffffu, mbar_wait(FE(slot), (nfr / NF - 1) & 1, failed, 540));
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
        }
        __syncwarp();
        ++nfr;
        if (!more) break;
        const int nt = f.j1 - f.j0;
        const int* row = p.table + static_cast<long long>(f.b) * p.width;
        float vr = 0.f;
        bool far = false;
        for (int t0 = 0; t0 < nt; t0 += NB) {
          const int key = (f.j0 + t0) * KT + 16 * lane;
          const bool live = key < f.len && key < f.j1 * KT;
          float ks = 0.f, vs = 1.f;
          bool good = true;
          if (live) {
            const int id = row[key >> p.block_log2];
            good = static_cast<unsigned>(id) < static_cast<unsigned>(p.N);
            if (good) {
              const long long cell = static_cast<long long>(id) * p.Hkv + f.kvh;
              ks = p.ks[cell] * p.scale_log2;
              vs = p.vs[cell];
            } else {
              ks = __int_as_float(0x7fc00000);
              record_error(7u, static_cast<unsigned>(f.b), static_cast<unsigned>(id));
            }
          }
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
          if (n_batch >= 2) ok = __all_sync(0xffffffffu, mbar_wait(SCE(bs), ((n_batch >> 1) - 1) & 1, failed, 541));
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
        }
        if (!ok) break;
      }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 14) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
  // The CTA that ends last leaves the tickets as they were.
  if (tid == 0 && atom_add_acq_rel_gpu(p.cnt + p.done, 1) == static_cast<int>(gridDim.x) - 1) {
    for (int i = 0; i < static_cast<int>(gridDim.x); ++i) p.cnt[i] = 0;
    p.cnt[p.done] = 0;
  }
}

}  // namespace du
