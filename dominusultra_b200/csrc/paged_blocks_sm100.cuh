// Blocks of the paged cache (layout in paged_sm100.cuh) that several requests share: forks, copies of
// blocks, and compaction.
//
// fork and compact work on sets of block ids. One cluster of eight CTAs finds out what happens: each CTA
// marks the ids of its share of the table in bitmaps of its own shared memory (atomics that stay on the
// SM), then takes a slice of the ids, joins that slice of the eight bitmaps over distributed shared memory,
// and what has to be numbered (free blocks, moves) is numbered by counting bits. Cluster barriers stand
// between the phases, and since sets and counts do not depend on the order of the marks, neither does any
// result.
//
// A call takes 10 to 18 us, all of it latency: loads that wait for loads, barriers, and the instructions' own
// way from L2, since a call runs through the code once (a fork of 64 requests, which takes 9.8 us now, took
// 12.6 with its loops unrolled, 42 KB of code instead of 21). Counts that all CTAs need are pushed into their
// shared memory before a barrier: pulled after it, eight CTAs' warps queued at one word for up to 2 us.
#pragma once

#include "du_ptx.cuh"

namespace du {

constexpr int PAGED_SET_CTAS = 8;  // the largest cluster that every device takes
constexpr int PAGED_SET_THREADS = 1024;
constexpr int PAGED_SET_WARPS = PAGED_SET_THREADS / 32;
constexpr int PAGED_SET_SMEM = 200 * 1024;  // bitmaps and per-request words
constexpr int PAGED_SET_PAGES = 128;        // table entries of a row that a warp takes at a time
constexpr int PAGED_APPLY_THREADS = 256;

__device__ __noinline__ void paged_set_error(unsigned code, unsigned a, unsigned b) { record_error(code, a, b); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// All threads of the cluster; writes before it, to shared and to global memory, are seen after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same in two parts. No CTA's shared memory may be touched by another before it runs, nor after it ends.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A word of another CTA's shared memory, at the address that it has in this one's.
__device__ __forceinline__ uint32_t cluster_load(const uint32_t* here, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ uint4 cluster_load4(const uint32_t* here, uint32_t rank) {
  uint32_t a;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_store2(const int2* here, uint32_t rank, int x, int y) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("st.shared::cluster.v2.s32 [%0], {%1, %2};" :: "r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void cluster_store1(const int* here, uint32_t rank, int x) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("st.shared::cluster.s32 [%0], %1;" :: "r"(a), "r"(x) : "memory");
}
// Bits taken out of a word of another CTA's.
__device__ __forceinline__ void cluster_and(const uint32_t* here, uint32_t rank, uint32_t mask) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.and.b32 [%0], %1;" :: "r"(a), "r"(mask) : "memory");
}
// A set of p.N ids as bits: words, and the share of them that a CTA joins (both whole 16-byte pieces).
__host__ __device__ __forceinline__ int set_words(int n) { return ((n + 127) >> 7) << 2; }
__host__ __device__ __forceinline__ int set_slice(int words) { return ((words + 4 * PAGED_SET_CTAS - 1) / (4 * PAGED_SET_CTAS)) * 4; }
// Words [w0, w1) of `sets` bitmaps of `words` words, joined over the eight CTAs into this one's. (The others
// read other words of this CTA's until the next cluster barrier.) All threads; four words each, a set
// after the other would wait for as many round trips.
__device__ __forceinline__ void join_slices(uint32_t* bits, int words, int sets, int w0, int w1) {
  const int pieces = (w1 - w0) >> 2;
#pragma unroll 1
  for (int i = threadIdx.x; i < sets * pieces; i += PAGED_SET_THREADS) {
    const int s = i >= 2 * pieces ? 2 : (i >= pieces ? 1 : 0);
    uint32_t* here = bits + s * words + w0 + 4 * (i - s * pieces);
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
      const uint4 v = cluster_load4(here, r);
      o.x |= v.x;
      o.y |= v.y;
      o.z |= v.z;
      o.w |= v.w;
    }
    *reinterpret_cast<uint4*>(here) = o;
  }
  __syncthreads();
}
// The ids below `end` of bits from word w0 on, the first of word w the rank[w - w0]-th, by put(rank, id).
template <typename Put>
__device__ __forceinline__ void list_bits(const uint32_t* bits, const int* rank, int w0, int end, Put put) {
#pragma unroll 4
  for (int id = 32 * w0 + static_cast<int>(threadIdx.x); id < end; id += PAGED_SET_THREADS) {
    const uint32_t m = bits[id >> 5], bit = 1u << (id & 31);
    if (m & bit) put(rank[(id >> 5) - w0] + __popc(m & (bit - 1u)), id);
  }
}

// Sum over the CTA of each thread's x; every thread gets the sum of all, and in `before` the sum over
// the threads below it. `part`: PAGED_SET_WARPS words of shared memory.
template <typename T>
__device__ __noinline__ T block_scan(T x, T* part, T& before) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T in = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T t = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += t;
  }
  __syncthreads();  // (part may still be read from the scan before)
  if (lane == 31) part[warp] = in;
  __syncthreads();
  T w = part[lane];  // (one word per warp: PAGED_SET_WARPS is 32)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  const T total = __shfl_sync(0xffffffffu, w, 31);
  const T below = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  before = in - x + (warp > 0 ? below : T(0));
  return total;
}
// Three counts in one word, for one scan (a set has fewer than 2^21 ids).
__device__ __forceinline__ unsigned long long count3(int a, int b, int c) {
  return static_cast<unsigned long long>(a) | static_cast<unsigned long long>(b) << 21 | static_cast<unsigned long long>(c) << 42;
}
__device__ __forceinline__ int count_of(unsigned long long n, int k) { return static_cast<int>(n >> (21 * k)) & 0x1fffff; }

static_assert(8LL * PAGED_SET_SMEM < 1 << 21, "count3");
static_assert(PAGED_SET_WARPS == 32, "block_scan takes one word per lane");

__device__ __forceinline__ void set_bit(uint32_t* bits, int id) { atomicOr(bits + (id >> 5), 1u << (id & 31)); }

// ---------------------------------------------------------------------------------------------
// Forks
// ---------------------------------------------------------------------------------------------
struct PagedForkParams {
  const int* table;    // [B, width]
  const int* lens;     // [B] tokens held
  const int* sources;  // [B] the request that b continues from
  const int* wanted;   // [B] tokens of it that b takes over
  int* ring;           // [N] free block ids, given back to in place
  const int* state;    // {head, count}
  int* table_out;      // [B, width]
  int* copies;         // [B, 2] {source block, destination block}, -1: none
  int* lens_out;       // [B]
  int* state_out;      // {head, count}
  int B, width, N, block, shift;  // tokens of a block, and their log2
};

// Slots of the hash table of B requests' last blocks, and the first one to look in for an id.
__host__ __device__ __forceinline__ int paged_fork_hash(int B) { return B + (B >> 1) + 1; }
__device__ __forceinline__ int paged_fork_slot(int id, int slots) {
  return static_cast<int>(__umulhi(static_cast<uint32_t>(id) * 2654435761u, static_cast<uint32_t>(slots)));
}
constexpr int PAGED_FORK_BLOCKS = (1 << 19) - 1;  // ids of 19 bits beside the requests' 13

// What request b takes over: the first `n` tokens of row `src`. A request with a length, source or
// wanted length out of range is kept: its row is copied as it is, and it holds its blocks whole. Where its own
// length is out of range nobody knows which of the row's entries are its blocks, so all that are block ids count
// as held after the call: others may share them, and none is given back. (They do not count as held before: a block
// that nobody else holds then stays out of the ring, as the row that names it stays.)
struct PagedForkAsk {
  int src, n;
  int pages, old_pages;  // blocks that it holds after and before
  bool kept, lost;       // lost: its own length is out of range
};
__device__ __forceinline__ PagedForkAsk paged_fork_ask(const PagedForkParams& p, int b) {
  PagedForkAsk a;
  const int cap = p.width * p.block;
  const int len = p.lens[b], s = p.sources[b], w = p.wanted[b];
  const bool own = len >= 0 && len <= cap;
  const bool from = s >= 0 && s < p.B;
  const int ls = p.lens[from ? s : b];
  a.lost = !own;
  a.kept = !own || !from || ls < 0 || ls > cap || w < 0 || w > ls;
  a.src = a.kept ? b : s;
  a.n = a.kept ? len : w;
  a.old_pages = own ? (len + p.block - 1) >> p.shift : 0;
  a.pages = a.lost ? p.width : (a.kept ? a.old_pages : (w + p.block - 1) >> p.shift);
  return a;
}

// Requests that continue from others, all at once from the state before the call.
//
// Row b becomes the first n_b tokens of row src_b; its whole blocks are shared. A last block that is
// partly filled will be written by b, so it has to be b's own: of the requests that hold it so, the
// lowest keeps it if no request holds it whole; the others get a free block each, in order of b from the
// ring's head, and a pair for paged_copy. One for which none is left is cut to its whole blocks. Blocks
// that some request held before and none holds after go behind the ring's tail, in order of their ids.
//
// With the sets O (held before), N (held after), W (held whole after): given back = O \ N, and b keeps
// its last block x iff x is not in W and no lower request ends partly in x. Marks are bits in shared
// memory; a warp takes 128 entries at a time, and its lanes fetch the lengths of 32 such pieces at once. The
// new rows are written while they are marked, all but the blocks that turn out to be the requests' own (written
// at the end, the rows cost a second pass: 8 us for 131072 entries, or the 4 us of a second launch). Whoever
// sees a partly filled last block tells all CTAs, and each finds the lowest request of every such block in a hash
// table of its own (entries {id, request} of 19 and 13 bits, the lowest stays).
//
// Bound by latency: chains of loads (source, length, entry; ring), two cluster barriers. 64 requests of
// 256 entries 9.8 us, 512 of 256 18.3 us.
__global__ void __cluster_dims__(PAGED_SET_CTAS, 1, 1) __launch_bounds__(PAGED_SET_THREADS, 1)
    paged_fork_kernel(const PagedForkParams p) {
  extern __shared__ __align__(16) uint32_t sm_set[];  // (taken in pieces of 16 bytes)
  __shared__ int part[PAGED_SET_WARPS];
  __shared__ int2 freed_of[PAGED_SET_CTAS];  // {ids given back in CTA r's slice, -}: each tells all
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int words = set_words(p.N), hashed = paged_fork_hash(p.B);
  uint32_t* before = sm_set;        // bits of the blocks held before
  uint32_t* after = before + words; // held after
  uint32_t* whole = after + words;  // held whole after
  int2* asked = reinterpret_cast<int2*>(whole + words);         // [B] {partly filled last block or -1, tokens; -1: kept}
  uint32_t* lowest = reinterpret_cast<uint32_t*>(asked + p.B);  // [hashed] {id, request}
#pragma unroll 1
  for (int i = tid; i < 3 * words; i += PAGED_SET_THREADS) sm_set[i] = 0u;
#pragma unroll 1
  for (int i = tid; i < hashed; i += PAGED_SET_THREADS) lowest[i] = 0xffffffffu;
  cluster_arrive();
  griddep_wait();
  const int head = p.state[0], count = p.state[1];
  bool ring_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;
  auto ring_at = [&](int i) { return head + i < p.N ? head + i : head + i - p.N; };  // (i <= N < 2^19)
  if (ring_ok && tid < min(p.B, count)) asm volatile("prefetch.global.L2 [%0];" :: "l"(p.ring + ring_at(tid)));

  // Marks. Pieces of rows: (request, 128 entries).
  const int per_row = (p.width + PAGED_SET_PAGES - 1) / PAGED_SET_PAGES;
  const int pieces = p.B * per_row;
  constexpr int all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const int share = (pieces + all_warps - 1) / all_warps;
  const int q_first = min((static_cast<int>(rank) * PAGED_SET_WARPS + warp) * share, pieces);
  const int q_end = min(q_first + share, pieces);
  bool all_here = false;  // the cluster's CTAs run
#pragma unroll 1
  for (int q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = min(32, q_end - q0);
    PagedForkAsk a{};
    const int my_b = (q0 + min(lane, nq - 1)) / per_row, my_c0 = (q0 + min(lane, nq - 1) - my_b * per_row) * PAGED_SET_PAGES;
    a = paged_fork_ask(p, my_b);
    if (a.kept && my_c0 == 0 && lane < nq) paged_set_error(6u, static_cast<unsigned>(my_b), static_cast<unsigned>(p.wanted[my_b]));
    // (a piece's entries are on their way while those of the one before are marked)
    int old_ids[PAGED_SET_PAGES / 32], new_ids[PAGED_SET_PAGES / 32];
    int b = 0, c0 = 0, pages = 0, partly = -1, tokens = 0, bad = 0;
    bool any_bad = false, lost = false;
#pragma unroll 1
    for (int i = 0; i <= nq; ++i) {
      int next_old[PAGED_SET_PAGES / 32], next_new[PAGED_SET_PAGES / 32];
      const int nb = __shfl_sync(0xffffffffu, my_b, i), nc0 = __shfl_sync(0xffffffffu, my_c0, i);
      const int src = __shfl_sync(0xffffffffu, a.src, i), n = __shfl_sync(0xffffffffu, a.n, i);
      const int npages = __shfl_sync(0xffffffffu, a.pages, i), old_pages = __shfl_sync(0xffffffffu, a.old_pages, i);
      const int how = __shfl_sync(0xffffffffu, static_cast<int>(a.kept) + static_cast<int>(a.lost), i);
      const bool kept = how != 0;
      if (i < nq) {
        const int* row_old = p.table + static_cast<long long>(nb) * p.width + nc0 + lane;
        const int* row_new = p.table + static_cast<long long>(src) * p.width + nc0 + lane;
        const int left_old = old_pages - nc0 - lane, left_new = (kept ? p.width : npages) - nc0 - lane;
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          next_old[k] = 32 * k < left_old ? row_old[32 * k] : -1;
          next_new[k] = 32 * k < left_new ? row_new[32 * k] : -1;
        }
      }
      if (i > 0) {
        int mine = -1;
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          const int page = c0 + 32 * k + lane, x = old_ids[k], y = new_ids[k];
          if (page < p.width) p.table_out[static_cast<long long>(b) * p.width + page] = y;
          if (page == partly) mine = y;
          if (static_cast<unsigned>(x) < static_cast<unsigned>(p.N)) set_bit(before, x);
          if (page < pages) {
            if (static_cast<unsigned>(y) < static_cast<unsigned>(p.N)) {
              set_bit(after, y);
              if (page != partly) set_bit(whole, y);
            } else if (!lost) {
              any_bad = true;
              bad = y;
            }
          }
        }
        const int at = max(partly, 0) - c0;  // (whoever has the partly filled block, or else the first entry, tells)
        if (at >= 0 && at < PAGED_SET_PAGES && (at & 31) == lane) {
          if (static_cast<unsigned>(mine) >= static_cast<unsigned>(p.N)) mine = -1;
#pragma unroll 1
          for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) cluster_store2(asked + b, r, mine, tokens);
        }
        if (any_bad) paged_set_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(bad));
        any_bad = false;
      } else if (!all_here) {
        cluster_wait();
        all_here = true;
      }
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        old_ids[k] = next_old[k];
        new_ids[k] = next_new[k];
      }
      b = nb;
      c0 = nc0;
      pages = npages;
      lost = how == 2;
      partly = !kept && (n & (p.block - 1)) != 0 ? npages - 1 : -1;
      tokens = kept ? -1 : n;
    }
  }
  if (!all_here) cluster_wait();
  cluster_sync();

  // The lowest request of each block that some end in.
#pragma unroll 1
  for (int b0 = 0; b0 < p.B; b0 += PAGED_SET_THREADS) {
    const int b = b0 + tid, x = b < p.B ? asked[b].x : -1;
    // (of the same block in a warp the lowest: requests from one prompt would queue at one slot)
    const uint32_t same = __match_any_sync(0xffffffffu, x);
    if (x < 0 || (same & ((1u << lane) - 1u))) continue;
    const uint32_t mine = static_cast<uint32_t>(x) << 13 | static_cast<uint32_t>(b);
#pragma unroll 1
    for (int i = paged_fork_slot(x, hashed);; i = i + 1 < hashed ? i + 1 : 0) {  // (more slots than requests: one is empty)
      const uint32_t there = atomicCAS(lowest + i, 0xffffffffu, mine);
      if (there == 0xffffffffu) break;
      if (there >> 13 == mine >> 13) {
        atomicMin(lowest + i, mine);
        break;
      }
    }
  }
  // This CTA's slice of the ids: the eight CTAs' bits joined, what nobody holds any more counted.
  const int slice = set_slice(words);
  const int w0 = min(static_cast<int>(rank) * slice, words), w1 = min(w0 + slice, words);
  join_slices(sm_set, words, 3, w0, w1);
  int gone = 0;
#pragma unroll 1
  for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) {
    before[w] &= ~after[w];
    gone += __popc(before[w]);
  }
  int below;
  const int gone_here = block_scan(gone, part, below);
  if (tid < PAGED_SET_CTAS) cluster_store2(freed_of + rank, static_cast<uint32_t>(tid), gone_here, 0);
  cluster_sync();

  const unsigned freed_there = lane < PAGED_SET_CTAS ? static_cast<unsigned>(freed_of[lane].x) : 0u;  // lane r: CTA r's
  const int freed = static_cast<int>(__reduce_add_sync(0xffffffffu, freed_there));
  const int freed_before = static_cast<int>(__reduce_add_sync(0xffffffffu, lane < static_cast<int>(rank) ? freed_there : 0u));
  // More given back than the ring has room for: the ring's state is not the tables'.
  if (static_cast<long long>(count) + freed > p.N) ring_ok = false;
  if (!ring_ok && rank == 0 && tid == 0) paged_set_error(7u, static_cast<unsigned>(head), static_cast<unsigned>(count));
  // Which requests need a block of their own, numbered in every CTA; CTA r's warps write each eighth warp's.
  int taken = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.B; b0 += PAGED_SET_THREADS) {
    const int b = b0 + tid;
    const int2 a = b < p.B ? asked[b] : make_int2(-1, 0);
    bool need = false;
    if (a.x >= 0) {
      const int w = a.x >> 5;
      need = (cluster_load(whole + w, static_cast<uint32_t>(w / slice)) >> (a.x & 31)) & 1u;
      int i = paged_fork_slot(a.x, hashed);
      while (lowest[i] >> 13 != static_cast<uint32_t>(a.x)) i = i + 1 < hashed ? i + 1 : 0;  // (it was put in)
      need = need || (lowest[i] & 8191u) != static_cast<uint32_t>(b);
    }
    int at;
    const int sum = block_scan(need ? 1 : 0, part, at);
    if (b < p.B && ((b >> 5) & (PAGED_SET_CTAS - 1)) == static_cast<int>(rank)) {
      int n = a.y, from = -1, own = -1;
      if (n < 0 || !ring_ok) {
        n = p.lens[b];
      } else if (need) {
        const int r = taken + at, last = ((n + p.block - 1) >> p.shift) - 1;
        if (r < count) {
          own = p.ring[ring_at(r)];
          from = a.x;
          if (static_cast<unsigned>(own) >= static_cast<unsigned>(p.N)) paged_set_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(own));
        } else {
          n = last * p.block;
        }
        p.table_out[static_cast<long long>(b) * p.width + last] = own;
      }
      p.lens_out[b] = n;
      p.copies[2LL * b] = from;
      p.copies[2LL * b + 1] = own;
    }
    taken += sum;
  }
  cluster_arrive();  // (nobody's shared memory is read from here on)
  taken = min(taken, count);
  if (!ring_ok) {  // every row as it was (the thread that wrote an entry writes it again)
#pragma unroll 1
    for (int q = q_first; q < q_end; ++q) {
      const int b = q / per_row, c0 = (q - b * per_row) * PAGED_SET_PAGES;
      for (int page = c0 + lane; page < min(c0 + PAGED_SET_PAGES, p.width); page += 32)
        p.table_out[static_cast<long long>(b) * p.width + page] = p.table[static_cast<long long>(b) * p.width + page];
    }
  } else {  // given back, behind the ring's tail
    int at = freed_before;
    int* rank_of = reinterpret_cast<int*>(after);  // (joined by all, by now)
#pragma unroll 1
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      int lower;
      const int sum = block_scan(w < w1 ? __popc(before[w]) : 0, part, lower);
      if (w < w1) rank_of[w - w0] = at + lower;
      at += sum;
    }
    __syncthreads();
    list_bits(before, rank_of, w0, 32 * w1, [&](int r, int id) { p.ring[ring_at(count + r)] = id; });
  }
  if (rank == 0 && tid == 0) {
    p.state_out[0] = ring_ok ? ring_at(taken) : head;
    p.state_out[1] = ring_ok ? count - taken + freed : count;
  }
  cluster_wait();
}

// Words of shared memory of a fork.
inline long long paged_fork_words(int B, int N) { return 3LL * set_words(N) + 2LL * B + paged_fork_hash(B); }

// ---------------------------------------------------------------------------------------------
// Compaction
// ---------------------------------------------------------------------------------------------
struct PagedCompactParams {
  const int* table;  // [B, width]
  const int* lens;   // [B] tokens held
  const int* ring;   // [N] free block ids
  const int* state;  // {head, count}
  int* table_out;    // [B, width]
  int* copies;       // [N / 2, 2] {source block, destination block}, -1: none
  int* ring_out;     // [N]
  int* state_out;    // {head, count}
  int4* map;         // for the second kernel: {end t, moves, in order?}, then for each 32 ids {those that move, moves
                     // before, those free afterwards, such before}
  int B, width, N, block, shift;  // tokens of a block, and their log2
};

// The requests' blocks moved to the lowest ids that they and the free blocks have between them.
//
// With U the ids in use, F the free ones, n = |U| and t the end of the lowest n of U + F: the ids of U
// from t on (there are as many as ids of F below t) move to the ids of F below t, the r-th to the r-th, in
// ascending order. The free ids are then those of U + F from t on, and the new ring holds them in
// ascending order from its start. Blocks that are in neither set belong to others and stay. A ring whose
// entries are not `count` different block ids that no request holds is not the tables': nothing moves.
//
// A request whose length is out of range keeps its row as it is, so none of the blocks in it may move, whoever else
// holds them: where there is such a request (every CTA is told), its entries are taken out of U again once U is
// joined, at the price of two more barriers.
//
// Ranks are counts of bits: of the slices before, of the words before in the slice, of the bits before in
// the word. The destinations are listed here, by rank; the second kernel looks a table's entry up by its
// rank, and lists sources and free ids.
//
// Bound by latency, as the fork; two cluster barriers. 16 requests of 64 entries 10.0 us, 256 of 512
// entries 17.7 us. The table's rows and the lists are written by a
// second launch over all SMs, whose CTAs are resident before the cluster ends: looking up 131072 entries
// took the cluster's eight SMs 20 us.
__global__ void __cluster_dims__(PAGED_SET_CTAS, 1, 1) __launch_bounds__(PAGED_SET_THREADS, 1)
    paged_compact_kernel(const PagedCompactParams p) {
  extern __shared__ __align__(16) uint32_t sm_set[];  // (taken in pieces of 16 bytes)
  __shared__ unsigned long long part[PAGED_SET_WARPS];
  __shared__ int2 told[2 * PAGED_SET_CTAS];  // {ids in use, free ids}, {ids that are both, -} of CTA r's slice: each tells all
  __shared__ int end_here[3];   // the end, ids in use and free ids before it in its slice
  __shared__ int lost;          // some request's length is out of range
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int words = set_words(p.N), slice = set_slice(words);
  uint32_t* used = sm_set;
  uint32_t* spare = used + words;
  int* rank_of = reinterpret_cast<int*>(spare + words);  // [slice] free ids below the end before each word of this slice
#pragma unroll 1
  for (int i = tid; i < 2 * words; i += PAGED_SET_THREADS) sm_set[i] = 0u;
  if (tid == 0) lost = 0;
  __syncwarp();
  cluster_arrive();
  griddep_launch_dependents();
  griddep_wait();
  const int head = p.state[0], count = p.state[1];
  const bool state_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;
  __syncthreads();

  // Marks.
  constexpr int threads = PAGED_SET_CTAS * PAGED_SET_THREADS;
  const int first = static_cast<int>(rank) * PAGED_SET_THREADS + tid;
  const int free_ids = state_ok ? count : 0;
  const int cap = p.width * p.block;
  const int per_row = (p.width + PAGED_SET_PAGES - 1) / PAGED_SET_PAGES;
  const int pieces = p.B * per_row;
  constexpr int all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const int share = (pieces + all_warps - 1) / all_warps;
  const int q_first = min((static_cast<int>(rank) * PAGED_SET_WARPS + warp) * share, pieces);
  const int q_end = min(q_first + share, pieces);
  bool any_lost = false;
#pragma unroll 1
  for (int q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = min(32, q_end - q0);
    const int my_b = (q0 + min(lane, nq - 1)) / per_row, my_c0 = (q0 + min(lane, nq - 1) - my_b * per_row) * PAGED_SET_PAGES;
    const int len = p.lens[my_b];
    const bool bad = len < 0 || len > cap;
    any_lost = any_lost || bad;
    if (bad && lane < nq) paged_set_error(6u, static_cast<unsigned>(my_b), static_cast<unsigned>(len));
    const int held = bad || lane >= nq ? 0 : (len + p.block - 1) >> p.shift;
    int ids[PAGED_SET_PAGES / 32], b = 0, left = 0, bad_id = 0;
    bool any_bad = false;
#pragma unroll 1
    for (int i = 0; i <= nq; ++i) {
      int next[PAGED_SET_PAGES / 32];
      const int nb = __shfl_sync(0xffffffffu, my_b, i), nc0 = __shfl_sync(0xffffffffu, my_c0, i);
      const int next_left = __shfl_sync(0xffffffffu, held, i) - nc0 - lane;
      if (i < nq) {
        const int* row = p.table + static_cast<long long>(nb) * p.width + nc0 + lane;
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) next[k] = 32 * k < next_left ? row[32 * k] : 0;
      }
      if (i > 0) {
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          if (32 * k >= left) continue;
          if (static_cast<unsigned>(ids[k]) < static_cast<unsigned>(p.N)) {
            set_bit(used, ids[k]);
          } else {
            any_bad = true;
            bad_id = ids[k];
          }
        }
        if (any_bad) paged_set_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(bad_id));
        any_bad = false;
      }
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) ids[k] = next[k];
      b = nb;
      left = next_left;
    }
  }
  constexpr int RING = 4;  // ids in flight
#pragma unroll 1
  for (int i0 = first; i0 < free_ids; i0 += RING * threads) {
    int ring[RING];
#pragma unroll
    for (int k = 0; k < RING; ++k) {
      const int i = i0 + threads * k;  // (below N + 2^16)
      ring[k] = i < free_ids ? p.ring[head + i < p.N ? head + i : head + i - p.N] : -1;
    }
#pragma unroll
    for (int k = 0; k < RING; ++k)
      if (static_cast<unsigned>(ring[k]) < static_cast<unsigned>(p.N)) set_bit(spare, ring[k]);
  }
  any_lost = __any_sync(0xffffffffu, any_lost);
  cluster_wait();  // (the cluster's CTAs run)
  if (any_lost && lane < PAGED_SET_CTAS) cluster_store1(&lost, static_cast<uint32_t>(lane), 1);
  cluster_sync();

  // This CTA's slice of the ids: the eight CTAs' bits joined and counted.
  const int w0 = min(static_cast<int>(rank) * slice, words), w1 = min(w0 + slice, words);
  join_slices(sm_set, words, 2, w0, w1);
  if (lost) {
    cluster_sync();
#pragma unroll 1
    for (int q = q_first; q < q_end; ++q) {
      const int b = q / per_row, c0 = (q - b * per_row) * PAGED_SET_PAGES, len = p.lens[b];
      if (len >= 0 && len <= cap) continue;
#pragma unroll 1
      for (int page = c0 + lane; page < min(c0 + PAGED_SET_PAGES, p.width); page += 32) {
        const int id = p.table[static_cast<long long>(b) * p.width + page];
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.N)) continue;
        const int w = id >> 5;
        const uint32_t owner = static_cast<uint32_t>(w / slice), bit = 1u << (id & 31);
        // (one that is in the ring too stays: the ring is not the tables' then)
        if (!(cluster_load(spare + w, owner) & bit)) cluster_and(used + w, owner, ~bit);
      }
    }
    __syncwarp();
    cluster_sync();
  }
  unsigned long long n3 = 0, below;
#pragma unroll 1
  for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) n3 += count3(__popc(used[w]), __popc(spare[w]), __popc(used[w] & spare[w]));
  n3 = block_scan(n3, part, below);
  if (tid < PAGED_SET_CTAS) {
    cluster_store2(told + 2 * rank, static_cast<uint32_t>(tid), count_of(n3, 0), count_of(n3, 1));
    cluster_store2(told + 2 * rank + 1, static_cast<uint32_t>(tid), count_of(n3, 2), 0);
  }
  cluster_sync();

  // (lane r of a warp has CTA r's)
  const bool one = lane < PAGED_SET_CTAS;
  const int of_used = one ? told[2 * lane].x : 0, of_spare = one ? told[2 * lane].y : 0, of_both = one ? told[2 * lane + 1].x : 0;
  const int all_used = __reduce_add_sync(0xffffffffu, of_used), all_spare = __reduce_add_sync(0xffffffffu, of_spare);
  const int all_both = __reduce_add_sync(0xffffffffu, of_both);
  const bool ok = state_ok && all_spare == count && all_both == 0;
  if (!ok && rank == 0 && tid == 0) paged_set_error(7u, static_cast<unsigned>(head), static_cast<unsigned>(count));
  // The slice in which the lowest all_used ids end, and how many of them it holds.
  int through = of_used + of_spare;
#pragma unroll
  for (int o = 1; o < PAGED_SET_CTAS; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, through, o);
    if (lane >= o) through += x;
  }
  const uint32_t reach = __ballot_sync(0xffffffffu, one && through >= all_used);  // (the last one does)
  const int end_slice = __ffs(static_cast<int>(reach)) - 1;
  const int rest = all_used - __shfl_sync(0xffffffffu, through - of_used - of_spare, end_slice);
  // Every CTA looks through that slice for the end, and for how many ids of either set lie before it there.
  const int e0 = min(end_slice * slice, words), e1 = min(e0 + slice, words);
  if (tid == 0) {
    end_here[0] = 32 * e0;
    end_here[1] = end_here[2] = 0;
  }
  unsigned long long seen = 0;
#pragma unroll 1
  for (int v0 = e0; v0 < e1; v0 += PAGED_SET_THREADS) {
    const int w = v0 + tid;
    const uint32_t u = w < e1 ? cluster_load(used + w, static_cast<uint32_t>(end_slice)) : 0u;
    const uint32_t f = w < e1 ? cluster_load(spare + w, static_cast<uint32_t>(end_slice)) : 0u;
    unsigned long long at;
    const unsigned long long sum = block_scan(count3(__popc(u), __popc(f), 0), part, at);
    at += seen;
    uint32_t m = u | f;
    int k = rest - count_of(at, 0) - count_of(at, 1);  // the k-th bit of this word is the last of the lowest
    if (k >= 1 && k <= __popc(m)) {
#pragma unroll 1
      for (; k > 1; --k) m &= m - 1u;
      const int last = __ffs(static_cast<int>(m));
      const uint32_t low = last == 32 ? 0xffffffffu : (1u << last) - 1u;
      end_here[0] = 32 * w + last;
      end_here[1] = count_of(at, 0) + __popc(u & low);
      end_here[2] = count_of(at, 1) + __popc(f & low);
    }
    seen += sum;
  }
  cluster_arrive();  // (nobody's shared memory is read from here on)
  __syncthreads();
  const int end = end_here[0];
  auto below_end = [&](int w) {
    const int d = end - 32 * w;
    return d <= 0 ? 0u : (d >= 32 ? 0xffffffffu : (1u << d) - 1u);
  };
  // Of each slice: moves, holes, free ids behind the end; all in the slices behind it, or before it, or parts.
  const int of_moves = lane > end_slice ? of_used : (lane == end_slice ? of_used - end_here[1] : 0);
  const int of_holes = lane < end_slice ? of_spare : (lane == end_slice ? end_here[2] : 0);
  const int of_left = lane > end_slice ? of_used + of_spare : (lane == end_slice ? of_used + of_spare - rest : 0);
  const bool lower = lane < static_cast<int>(rank);
  const int all_moves = __reduce_add_sync(0xffffffffu, of_moves);
  int moves = __reduce_add_sync(0xffffffffu, lower ? of_moves : 0), holes = __reduce_add_sync(0xffffffffu, lower ? of_holes : 0);
  int left = __reduce_add_sync(0xffffffffu, lower ? of_left : 0);
  if (rank == 0 && tid == 0) {
    p.map[0] = make_int4(end, ok ? all_moves : 0, ok, count);
    p.state_out[0] = ok ? 0 : head;
    p.state_out[1] = count;
  }
  if (ok) {
#pragma unroll 1
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      const uint32_t low = below_end(w);
      const uint32_t u = w < w1 ? used[w] : 0u, f = w < w1 ? spare[w] : 0u;
      const unsigned long long sum = block_scan(count3(__popc(u & ~low), __popc(f & low), __popc((u | f) & ~low)), part, below);
      if (w < w1) {
        p.map[1 + w] = make_int4(static_cast<int>(u & ~low), moves + count_of(below, 0), static_cast<int>((u | f) & ~low), left + count_of(below, 2));
        rank_of[w - w0] = holes + count_of(below, 1);
      }
      moves += count_of(sum, 0);
      holes += count_of(sum, 1);
      left += count_of(sum, 2);
    }
    __syncthreads();
    list_bits(spare, rank_of, w0, min(32 * w1, end), [&](int r, int id) { p.copies[2LL * r + 1] = id; });
  }
  cluster_wait();
}

// The compaction's rows (an entry per thread), sources and free ids (an id per thread).
__global__ void __launch_bounds__(PAGED_APPLY_THREADS) paged_compact_rows_kernel(const PagedCompactParams p) {
  griddep_wait();
  const unsigned first = blockIdx.x * PAGED_APPLY_THREADS + threadIdx.x, step = gridDim.x * PAGED_APPLY_THREADS;
  const int4 h = __ldcg(p.map);
  const int end = h.x, moves = h.y, count = h.w;
  const bool ok = h.z != 0;
  const int cap = p.width * p.block;
  const unsigned entries = static_cast<unsigned>(p.B) * static_cast<unsigned>(p.width);
  for (unsigned e = first; e < entries; e += step) {
    const unsigned b = e / static_cast<unsigned>(p.width);
    const int page = static_cast<int>(e - b * static_cast<unsigned>(p.width));
    const int len = p.lens[b];
    int x = p.table[e];
    if (ok && len >= 0 && len <= cap) {
      if (page >= (len + p.block - 1) >> p.shift) {
        x = -1;
      } else if (x >= end && x < p.N) {
        const int4 m = __ldcg(p.map + 1 + (x >> 5));
        const uint32_t bit = 1u << (x & 31);
        if (static_cast<uint32_t>(m.x) & bit)  // (else it stays)
          x = __ldcg(p.copies + 2LL * (m.y + __popc(static_cast<uint32_t>(m.x) & (bit - 1u))) + 1);
      }
    }
    p.table_out[e] = x;
  }
  for (unsigned i = first; i < static_cast<unsigned>(p.N); i += step) {
    const int id = static_cast<int>(i);
    if (!ok) {
      p.ring_out[id] = p.ring[id];
    } else {
      const int4 m = __ldcg(p.map + 1 + (id >> 5));
      const uint32_t bit = 1u << (id & 31);
      if (static_cast<uint32_t>(m.x) & bit) p.copies[2LL * (m.y + __popc(static_cast<uint32_t>(m.x) & (bit - 1u)))] = id;
      if (static_cast<uint32_t>(m.z) & bit) p.ring_out[m.w + __popc(static_cast<uint32_t>(m.z) & (bit - 1u))] = id;
      if (id >= count) p.ring_out[id] = -1;
    }
    if (id >= moves && id < p.N / 2) {
      p.copies[2LL * id] = -1;
      p.copies[2LL * id + 1] = -1;
    }
  }
}

// Bytes of workspace of a compaction.
inline size_t paged_compact_ws(int N) { return sizeof(int4) * static_cast<size_t>(1 + set_words(N)); }

// Words of shared memory of a compaction.
inline long long paged_compact_words(int N) { return 2LL * set_words(N) + set_slice(set_words(N)); }
constexpr int PAGED_COMPACT_BLOCKS = 770000;  // (what fits PAGED_SET_SMEM; du_paged_compact checks the words too)

// ---------------------------------------------------------------------------------------------
// Copies
// ---------------------------------------------------------------------------------------------
struct PagedCopyParams {
  uint8_t* k8;        // [N, Hkv, block, D] e4m3
  uint8_t* v8;
  float* ks;          // [N, Hkv]
  float* vs;
  const int* copies;  // [n, 2] {source block, destination block}, -1: none
  int n, N, Hkv;
  long long bytes;    // of a block in one cache, a multiple of 256
  int parts;          // of PAGED_COPY_PART bytes
};
constexpr int PAGED_COPY_PART = 2048;  // bytes that a warp takes at a time: four 16-byte loads per lane
constexpr int PAGED_COPY_THREADS = 256;

// Copies of blocks within a cache: keys, values and their scales. A warp takes 2 KB of a block, so that its
// loads are in flight together and one block is spread over several warps; bound by HBM (every byte read and
// written once): 4096 blocks of 32 tokens, 8 heads of 128, 84 us, 5.8 TB/s, 0.9 of a plain copy; 64 pairs 2.7 us.
__global__ void __launch_bounds__(PAGED_COPY_THREADS) paged_copy_kernel(const PagedCopyParams p) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (PAGED_COPY_THREADS / 32);
  const long long items = 2LL * p.n * p.parts;
  griddep_wait();
  for (long long it = (static_cast<long long>(blockIdx.x) * PAGED_COPY_THREADS + threadIdx.x) >> 5; it < items; it += warps) {
    const long long pair = it / (2 * p.parts);
    const int rest = static_cast<int>(it - pair * 2 * p.parts);
    const bool values = rest >= p.parts;
    const int part = values ? rest - p.parts : rest;
    const int2 c = make_int2(p.copies[2 * pair], p.copies[2 * pair + 1]);
    if (c.x == -1 && c.y == -1) continue;
    if (static_cast<unsigned>(c.x) >= static_cast<unsigned>(p.N) || static_cast<unsigned>(c.y) >= static_cast<unsigned>(p.N)) {
      if (lane == 0 && rest == 0)
        record_error(7u, static_cast<unsigned>(pair), static_cast<unsigned>(static_cast<unsigned>(c.x) >= static_cast<unsigned>(p.N) ? c.x : c.y));
      continue;
    }
    uint8_t* cache = values ? p.v8 : p.k8;
    const long long off = static_cast<long long>(part) * PAGED_COPY_PART + 16 * lane;
    const uint8_t* src = cache + c.x * p.bytes + off;
    uint8_t* dst = cache + c.y * p.bytes + off;
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (off + 512 * i < p.bytes) x[i] = *reinterpret_cast<const uint4*>(src + 512 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (off + 512 * i < p.bytes) *reinterpret_cast<uint4*>(dst + 512 * i) = x[i];
    if (part == 0) {
      float* s = values ? p.vs : p.ks;
      for (int h = lane; h < p.Hkv; h += 32) s[static_cast<long long>(c.y) * p.Hkv + h] = s[static_cast<long long>(c.x) * p.Hkv + h];
    }
  }
}

}  // namespace du
