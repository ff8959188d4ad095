// Blocks of the paged cache (layout in paged_sm100.cuh) that several requests share: forks, copies of
// blocks, and compaction.
//
// fork and compact work on sets of block ids. One cluster of eight CTAs finds out what happens: each CTA
// marks the ids of its share of the table in bitmaps of its own shared memory (atomics that stay on the
// SM), then takes a slice of the ids, joins that slice of the eight bitmaps over distributed shared memory,
// and what has to be numbered (free blocks, moves) is numbered by counting bits. Cluster barriers stand
// between the phases, and since sets and counts do not depend on the order of the marks, neither does any
// result.
#pragma once

#include "du_ptx.cuh"

namespace du {

constexpr int PAGED_SET_CTAS = 8;  // the largest cluster that every device takes
constexpr int PAGED_SET_THREADS = 1024;
constexpr int PAGED_SET_WARPS = PAGED_SET_THREADS / 32;
constexpr int PAGED_SET_SMEM = 200 * 1024;  // bitmaps and per-request words
constexpr int PAGED_SET_PAGES = 128;        // table entries of a row that a warp takes at a time
constexpr int PAGED_APPLY_THREADS = 256;

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
// The same in two parts, for the end: no CTA may leave while another still reads its shared memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A word of another CTA's shared memory, at the address that it has in this one's.
__device__ __forceinline__ uint32_t cluster_load(const uint32_t* here, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Sum over the CTA of each thread's x; every thread gets the sum of all, and in `before` the sum over
// the threads below it. `part`: PAGED_SET_WARPS words of shared memory.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* part, T& before) {
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
// Three counts of bits in one word, for one scan (a set has fewer than 2^21 ids).
__device__ __forceinline__ unsigned long long count3(uint32_t a, uint32_t b, uint32_t c) {
  return static_cast<unsigned long long>(__popc(a)) | static_cast<unsigned long long>(__popc(b)) << 21 | static_cast<unsigned long long>(__popc(c)) << 42;
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
  int B, width, N, block;
};

// What request b takes over: the first `n` tokens of row `src`. A request with a length, source or
// wanted length out of range is kept: its row is copied as it is, and it holds its blocks whole (none,
// if its own length is out of range).
struct PagedForkAsk {
  int src, n;
  int pages, old_pages;  // blocks that it holds after and before
  bool kept;
};
__device__ __forceinline__ PagedForkAsk paged_fork_ask(const PagedForkParams& p, int b) {
  PagedForkAsk a;
  const int cap = p.width * p.block;
  const int len = p.lens[b], s = p.sources[b], w = p.wanted[b];
  const bool own = len >= 0 && len <= cap;
  const bool from = s >= 0 && s < p.B;
  const int ls = p.lens[from ? s : b];
  a.kept = !own || !from || ls < 0 || ls > cap || w < 0 || w > ls;
  a.src = a.kept ? b : s;
  a.n = a.kept ? len : w;
  a.old_pages = own ? (len + p.block - 1) / p.block : 0;
  a.pages = a.kept ? a.old_pages : (w + p.block - 1) / p.block;
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
// memory; a warp takes two pieces of 128 entries at a time, and its lanes fetch the lengths of 32 such
// pieces at once. The new rows are written while they are marked, all but the blocks that turn out to be
// the requests' own (written at the end, the rows cost a second pass: 8 us for 131072 entries, or the
// 4 us of a second launch). The lowest request is found by comparing the last blocks of those before it, 32 at a time.
//
// Bound by latency: chains of loads (source, length, entry; ring), four cluster barriers.
__global__ void __cluster_dims__(PAGED_SET_CTAS, 1, 1) __launch_bounds__(PAGED_SET_THREADS, 1)
    paged_fork_kernel(const PagedForkParams p) {
  extern __shared__ uint32_t sm_set[];
  __shared__ int part[PAGED_SET_WARPS];
  __shared__ uint32_t freed_here;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int words = (p.N + 31) >> 5, flags = (p.B + 31) >> 5;
  uint32_t* before = sm_set;                // bits of the blocks held before
  uint32_t* after = before + words;         // held after
  uint32_t* whole = after + words;          // held whole after
  uint32_t* needs = whole + words;          // [flags] bits of the requests that need a block: this CTA's
  uint32_t* needs_all = needs + flags;      // [flags] and all of them
  int* need_rank = reinterpret_cast<int*>(needs_all + flags);  // [flags] needs before each 32 requests
  int* last = need_rank + flags;            // [B] a partly filled last block, else -1
  for (int i = tid; i < 3 * words + flags; i += PAGED_SET_THREADS) sm_set[i] = 0u;
  griddep_launch_dependents();
  griddep_wait();
  const int head = p.state[0], count = p.state[1];
  bool ring_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;
  for (int b = tid; b < p.B; b += PAGED_SET_THREADS) {
    const PagedForkAsk a = paged_fork_ask(p, b);
    int id = -1;
    if (!a.kept && a.n % p.block != 0) {
      id = p.table[static_cast<long long>(a.src) * p.width + a.pages - 1];
      if (id >= p.N) id = -1;
    }
    last[b] = id;
    if (a.kept && rank == 0) record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(p.wanted[b]));
  }
  __syncthreads();

  // Marks. Pieces of rows: (request, 128 entries).
  const int per_row = (p.width + PAGED_SET_PAGES - 1) / PAGED_SET_PAGES;
  const int pieces = p.B * per_row;
  constexpr int all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const int share = (pieces + all_warps - 1) / all_warps;
  const int q_first = min((static_cast<int>(rank) * PAGED_SET_WARPS + warp) * share, pieces);
  const int q_end = min(q_first + share, pieces);
  for (int q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = min(32, q_end - q0);
    PagedForkAsk a{};
    const int my_b = (q0 + min(lane, nq - 1)) / per_row, my_c0 = (q0 + min(lane, nq - 1) - my_b * per_row) * PAGED_SET_PAGES;
    a = paged_fork_ask(p, my_b);
    for (int i = 0; i < nq; i += 2) {
      int ids[2][2][PAGED_SET_PAGES / 32], b[2], c0[2], pages[2], partly[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int from = min(i + h, nq - 1);
        b[h] = __shfl_sync(0xffffffffu, my_b, from);
        c0[h] = __shfl_sync(0xffffffffu, my_c0, from);
        const int src = __shfl_sync(0xffffffffu, a.src, from);
        const int n = __shfl_sync(0xffffffffu, a.n, from);
        pages[h] = __shfl_sync(0xffffffffu, a.pages, from);
        int old_pages = __shfl_sync(0xffffffffu, a.old_pages, from);
        const bool kept = __shfl_sync(0xffffffffu, static_cast<int>(a.kept), from) != 0;
        partly[h] = !kept && n % p.block != 0 ? pages[h] - 1 : -1;
        if (i + h >= nq) pages[h] = old_pages = 0;
        const int* row_old = p.table + static_cast<long long>(b[h]) * p.width;
        const int* row_new = p.table + static_cast<long long>(src) * p.width;
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          const int page = c0[h] + 32 * k + lane;
          ids[h][0][k] = page < old_pages ? row_old[page] : -1;
          ids[h][1][k] = page < (kept ? (i + h < nq ? p.width : 0) : pages[h]) ? row_new[page] : -1;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          const int page = c0[h] + 32 * k + lane;
          const int x = ids[h][0][k], y = ids[h][1][k];
          if (page < p.width && i + h < nq) p.table_out[static_cast<long long>(b[h]) * p.width + page] = y;
          if (static_cast<unsigned>(x) < static_cast<unsigned>(p.N)) set_bit(before, x);
          if (page < pages[h]) {
            if (static_cast<unsigned>(y) < static_cast<unsigned>(p.N)) {
              set_bit(after, y);
              if (page != partly[h]) set_bit(whole, y);
            } else {
              record_error(7u, static_cast<unsigned>(b[h]), static_cast<unsigned>(y));
            }
          }
        }
      }
    }
  }
  cluster_sync();

  // This CTA's slice of the ids: the eight CTAs' bits joined, what nobody holds any more counted.
  const int slice = (words + PAGED_SET_CTAS - 1) / PAGED_SET_CTAS;
  const int w0 = min(static_cast<int>(rank) * slice, words), w1 = min(w0 + slice, words);
  int gone = 0;
  for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) {
    uint32_t o = 0u, n = 0u, f = 0u;
#pragma unroll
    for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
      o |= cluster_load(before + w, r);
      n |= cluster_load(after + w, r);
      f |= cluster_load(whole + w, r);
    }
    // (other CTAs read other slices of this CTA's bitmaps until the next barrier)
    before[w] = o & ~n;
    whole[w] = f;
    gone += __popc(o & ~n);
  }
  int below;
  const int gone_here = block_scan(gone, part, below);
  if (tid == 0) freed_here = static_cast<uint32_t>(gone_here);
  cluster_sync();

  // Which requests of this CTA's share need a block of their own.
  for (int b = static_cast<int>(rank) * PAGED_SET_WARPS + warp; b < p.B; b += PAGED_SET_CTAS * PAGED_SET_WARPS) {
    const int x = last[b];
    if (x < 0) continue;
    const int w = x >> 5;
    bool need = (cluster_load(whole + w, static_cast<uint32_t>(w / slice)) >> (x & 31)) & 1u;
    for (int c = 0; c < b && !need; c += 32) need = __any_sync(0xffffffffu, c + lane < b && last[c + lane] == x);
    if (need && lane == 0) atomicOr(needs + (b >> 5), 1u << (b & 31));
  }
  int freed = 0, freed_before = 0;
#pragma unroll
  for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
    const int n = static_cast<int>(cluster_load(&freed_here, r));
    if (r < rank) freed_before += n;
    freed += n;
  }
  // More given back than the ring has room for: the ring's state is not the tables'.
  if (static_cast<long long>(count) + freed > p.N) ring_ok = false;
  if (!ring_ok && rank == 0 && tid == 0) record_error(7u, static_cast<unsigned>(head), static_cast<unsigned>(count));
  cluster_sync();

  // Every CTA: all the requests' flags, and how many needs lie before each 32 of them.
  int taken = 0;
  for (int i0 = 0; i0 < flags; i0 += PAGED_SET_THREADS) {
    const int i = i0 + tid;
    uint32_t m = 0u;
    if (i < flags) {
#pragma unroll
      for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) m |= cluster_load(needs + i, r);
    }
    int at;
    const int sum = block_scan(__popc(m), part, at);
    if (i < flags) {
      need_rank[i] = taken + at;
      needs_all[i] = m;
    }
    taken += sum;
  }
  __syncthreads();
  cluster_arrive();  // (nobody's shared memory is read from here on)
  taken = min(taken, count);
  auto ring_at = [&](int i) { return head + i < p.N ? head + i : head + i - p.N; };  // (i <= N < 2^21)
  // Requests: CTA r takes every eighth from the r-th on.
  for (int b = PAGED_SET_CTAS * tid + static_cast<int>(rank); b < p.B; b += PAGED_SET_CTAS * PAGED_SET_THREADS) {
    const PagedForkAsk a = paged_fork_ask(p, b);
    const bool kept = a.kept || !ring_ok;
    int n = kept ? p.lens[b] : a.n, from = -1, own = -1;
    const uint32_t m = needs_all[b >> 5];
    if (!kept && ((m >> (b & 31)) & 1u)) {
      const int r = need_rank[b >> 5] + __popc(m & ((1u << (b & 31)) - 1u));
      if (r < count) {
        own = p.ring[ring_at(r)];
        from = last[b];
        if (static_cast<unsigned>(own) >= static_cast<unsigned>(p.N)) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(own));
      } else {
        n = (a.pages - 1) * p.block;
      }
      p.table_out[static_cast<long long>(b) * p.width + a.pages - 1] = own;
    }
    p.lens_out[b] = n;
    p.copies[2LL * b] = from;
    p.copies[2LL * b + 1] = own;
  }
  if (!ring_ok) {  // every row as it was (the thread that wrote an entry writes it again)
    for (int q = q_first; q < q_end; ++q) {
      const int b = q / per_row, c0 = (q - b * per_row) * PAGED_SET_PAGES;
      for (int page = c0 + lane; page < min(c0 + PAGED_SET_PAGES, p.width); page += 32)
        p.table_out[static_cast<long long>(b) * p.width + page] = p.table[static_cast<long long>(b) * p.width + page];
    }
  }
  // Given back, behind the ring's tail: a warp's words one by one, a bit per lane.
  if (ring_ok) {
    int at = freed_before;
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      const uint32_t m = w < w1 ? before[w] : 0u;
      int lower;
      const int sum = block_scan(__popc(m), part, lower);
      for (uint32_t any = __ballot_sync(0xffffffffu, m != 0u); any; any &= any - 1u) {
        const int j = __ffs(static_cast<int>(any)) - 1;
        const uint32_t word = __shfl_sync(0xffffffffu, m, j);
        const int i = at + __shfl_sync(0xffffffffu, lower, j) + __popc(word & ((1u << lane) - 1u));
        if ((word >> lane) & 1u) p.ring[ring_at(count + i)] = 32 * (w - lane + j) + lane;
      }
      at += sum;
    }
  }
  if (rank == 0 && tid == 0) {
    p.state_out[0] = ring_ok ? ring_at(taken) : head;
    p.state_out[1] = ring_ok ? count - taken + freed : count;
  }
  cluster_wait();
}

// Words of shared memory of a fork.
inline long long paged_fork_words(long long B, long long N) { return 3 * ((N + 31) / 32) + 3 * ((B + 31) / 32) + B; }

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
  int B, width, N, block;
};

// The requests' blocks moved to the lowest ids that they and the free blocks have between them.
//
// With U the ids in use, F the free ones, n = |U| and t the end of the lowest n of U + F: the ids of U
// from t on (there are as many as ids of F below t) move to the ids of F below t, the r-th to the r-th, in
// ascending order. The free ids are then those of U + F from t on, and the new ring holds them in
// ascending order from its start. Blocks that are in neither set belong to others and stay. A ring whose
// entries are not `count` different block ids that no request holds is not the tables': nothing moves.
//
// Ranks are counts of bits: of the slices before, of the words before in the slice, of the bits before in
// the word. The destinations are listed here, by rank; the second kernel looks a table's entry up by its
// rank, and lists sources and free ids.
//
// Bound by latency, as the fork; three cluster barriers. The table's rows and the lists are written by a
// second launch over all SMs, whose CTAs are resident before the cluster ends: looking up 131072 entries
// took the cluster's eight SMs 20 us.
__global__ void __cluster_dims__(PAGED_SET_CTAS, 1, 1) __launch_bounds__(PAGED_SET_THREADS, 1)
    paged_compact_kernel(const PagedCompactParams p) {
  extern __shared__ uint32_t sm_set[];
  __shared__ unsigned long long part[PAGED_SET_WARPS];
  __shared__ uint32_t told[3];  // of this CTA's slice: ids in use, free ids, ids that are both
  __shared__ int end_here;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int words = (p.N + 31) >> 5;
  const int slice = (words + PAGED_SET_CTAS - 1) / PAGED_SET_CTAS;
  uint32_t* used = sm_set;
  uint32_t* spare = used + words;
  for (int i = tid; i < 2 * words; i += PAGED_SET_THREADS) sm_set[i] = 0u;
  griddep_launch_dependents();
  griddep_wait();
  const int head = p.state[0], count = p.state[1];
  const bool state_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;
  __syncthreads();

  // Marks: the ring's ids are fetched before the table's and marked after them.
  constexpr int threads = PAGED_SET_CTAS * PAGED_SET_THREADS;
  const int first = static_cast<int>(rank) * PAGED_SET_THREADS + tid;
  const int free_ids = state_ok ? count : 0;
  constexpr int RING = 8;
  int ring[RING];
  auto ring_load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < RING; ++k) {
      const int i = i0 + threads * k;  // (below N + 2^16)
      ring[k] = i < free_ids ? p.ring[head + i < p.N ? head + i : head + i - p.N] : -1;
    }
  };
  auto ring_mark = [&]() {
#pragma unroll
    for (int k = 0; k < RING; ++k)
      if (static_cast<unsigned>(ring[k]) < static_cast<unsigned>(p.N)) set_bit(spare, ring[k]);
  };
  ring_load(first);
  const int cap = p.width * p.block;
  const int per_row = (p.width + PAGED_SET_PAGES - 1) / PAGED_SET_PAGES;
  const int pieces = p.B * per_row;
  constexpr int all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const int share = (pieces + all_warps - 1) / all_warps;
  const int q_first = min((static_cast<int>(rank) * PAGED_SET_WARPS + warp) * share, pieces);
  const int q_end = min(q_first + share, pieces);
  for (int q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = min(32, q_end - q0);
    const int my_b = (q0 + min(lane, nq - 1)) / per_row, my_c0 = (q0 + min(lane, nq - 1) - my_b * per_row) * PAGED_SET_PAGES;
    const int len = p.lens[my_b];
    const bool bad = len < 0 || len > cap;
    if (bad && lane < nq) record_error(6u, static_cast<unsigned>(my_b), static_cast<unsigned>(len));
    const int held = bad || lane >= nq ? 0 : (len + p.block - 1) / p.block;
    for (int i = 0; i < nq; i += 2) {
      int ids[2][PAGED_SET_PAGES / 32], b[2], c0[2], n[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        b[h] = __shfl_sync(0xffffffffu, my_b, i + h);
        c0[h] = __shfl_sync(0xffffffffu, my_c0, i + h);
        n[h] = __shfl_sync(0xffffffffu, held, i + h);  // (0 behind the last piece: i is even, so lane i + h exists)
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          const int page = c0[h] + 32 * k + lane;
          ids[h][k] = page < n[h] ? p.table[static_cast<long long>(b[h]) * p.width + page] : 0;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
          if (c0[h] + 32 * k + lane >= n[h]) continue;
          if (static_cast<unsigned>(ids[h][k]) < static_cast<unsigned>(p.N)) set_bit(used, ids[h][k]);
          else record_error(7u, static_cast<unsigned>(b[h]), static_cast<unsigned>(ids[h][k]));
        }
      }
    }
  }
  ring_mark();
  for (int i0 = first + RING * threads; i0 < free_ids; i0 += RING * threads) {
    ring_load(i0);
    ring_mark();
  }
  cluster_sync();

  // This CTA's slice of the ids: the eight CTAs' bits joined and counted.
  const int w0 = min(static_cast<int>(rank) * slice, words), w1 = min(w0 + slice, words);
  unsigned long long n3 = 0, below;
  for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) {
    uint32_t u = 0u, f = 0u;
#pragma unroll
    for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
      u |= cluster_load(used + w, r);
      f |= cluster_load(spare + w, r);
    }
    // (other CTAs read other slices of this CTA's bitmaps until the next barrier)
    used[w] = u;
    spare[w] = f;
    n3 += count3(u, f, u & f);
  }
  n3 = block_scan(n3, part, below);
  if (tid < 3) told[tid] = static_cast<uint32_t>(count_of(n3, tid));
  cluster_sync();

  int all_used = 0, all_spare = 0, all_both = 0;
  int of_used[PAGED_SET_CTAS], of_spare[PAGED_SET_CTAS];
#pragma unroll
  for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
    of_used[r] = static_cast<int>(cluster_load(told, r));
    of_spare[r] = static_cast<int>(cluster_load(told + 1, r));
    all_used += of_used[r];
    all_spare += of_spare[r];
    all_both += static_cast<int>(cluster_load(told + 2, r));
  }
  const bool ok = state_ok && all_spare == count && all_both == 0;
  if (!ok && rank == 0 && tid == 0) record_error(7u, static_cast<unsigned>(head), static_cast<unsigned>(count));
  // The slice in which the lowest all_used ids end, and how many of them it holds.
  int end_slice = -1, rest = all_used;
#pragma unroll
  for (int r = 0; r < PAGED_SET_CTAS; ++r) {
    if (end_slice < 0) {
      if (rest <= of_used[r] + of_spare[r]) end_slice = r;
      else rest -= of_used[r] + of_spare[r];
    }
  }
  if (end_slice < 0) end_slice = PAGED_SET_CTAS - 1;  // (out of reach: the slices hold all_used ids and more)
  // Every CTA looks through that slice for the end, and counts its ids in use above and its free ids below
  // the end (by counting those below, in two of the fields).
  const int e0 = min(end_slice * slice, words), e1 = min(e0 + slice, words);
  if (tid == 0) end_here = 32 * e0;
  int seen = 0;
  for (int v0 = e0; v0 < e1; v0 += PAGED_SET_THREADS) {
    const int w = v0 + tid;
    uint32_t m = w < e1 ? cluster_load(used + w, static_cast<uint32_t>(end_slice)) | cluster_load(spare + w, static_cast<uint32_t>(end_slice)) : 0u;
    unsigned long long at;
    const int c = __popc(m), sum = static_cast<int>(block_scan(static_cast<unsigned long long>(c), part, at));
    int k = rest - seen - static_cast<int>(at);  // the k-th bit of this word is the last of the lowest
    if (k >= 1 && k <= c) {
      for (; k > 1; --k) m &= m - 1u;
      end_here = 32 * w + __ffs(static_cast<int>(m));
    }
    seen += sum;
  }
  __syncthreads();
  const int end = end_here;
  auto below_end = [&](int w) {
    const int d = end - 32 * w;
    return d <= 0 ? 0u : (d >= 32 ? 0xffffffffu : (1u << d) - 1u);
  };
  n3 = 0;
  for (int w = e0 + tid; w < e1; w += PAGED_SET_THREADS) {
    const uint32_t low = below_end(w);
    n3 += count3(cluster_load(used + w, static_cast<uint32_t>(end_slice)) & ~low, cluster_load(spare + w, static_cast<uint32_t>(end_slice)) & low, 0u);
  }
  cluster_arrive();  // (nobody's shared memory is read from here on)
  n3 = block_scan(n3, part, below);
  const int end_moves = count_of(n3, 0), end_holes = count_of(n3, 1);
  int all_moves = end_moves, moves = 0, holes = 0, left = 0;
#pragma unroll
  for (int r = 0; r < PAGED_SET_CTAS; ++r) {
    if (r > end_slice) all_moves += of_used[r];
    if (r >= static_cast<int>(rank)) continue;
    moves += r == end_slice ? end_moves : (r > end_slice ? of_used[r] : 0);
    holes += r == end_slice ? end_holes : (r < end_slice ? of_spare[r] : 0);
    left += r == end_slice ? of_used[r] + of_spare[r] - rest : (r > end_slice ? of_used[r] + of_spare[r] : 0);
  }
  if (rank == 0 && tid == 0) {
    p.map[0] = make_int4(end, ok ? all_moves : 0, ok, count);
    p.state_out[0] = ok ? 0 : head;
    p.state_out[1] = count;
  }
  if (ok) {
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      const uint32_t low = below_end(w);
      const uint32_t u = w < w1 ? used[w] : 0u, f = w < w1 ? spare[w] : 0u;
      const uint32_t hole = f & low;
      const unsigned long long sum = block_scan(count3(u & ~low, hole, (u | f) & ~low), part, below);
      if (w < w1)
        p.map[1 + w] = make_int4(static_cast<int>(u & ~low), moves + count_of(below, 0), static_cast<int>((u | f) & ~low), left + count_of(below, 2));
      const int at = holes + count_of(below, 1);
      for (uint32_t any = __ballot_sync(0xffffffffu, hole != 0u); any; any &= any - 1u) {
        const int j = __ffs(static_cast<int>(any)) - 1;
        const uint32_t word = __shfl_sync(0xffffffffu, hole, j);
        const int r = __shfl_sync(0xffffffffu, at, j) + __popc(word & ((1u << lane) - 1u));
        if ((word >> lane) & 1u) p.copies[2LL * r + 1] = 32 * (w - lane + j) + lane;
      }
      moves += count_of(sum, 0);
      holes += count_of(sum, 1);
      left += count_of(sum, 2);
    }
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
      if (page >= (len + p.block - 1) / p.block) {
        x = -1;
      } else if (x >= end && x < p.N) {
        const int4 m = __ldcg(p.map + 1 + (x >> 5));
        x = __ldcg(p.copies + 2LL * (m.y + __popc(static_cast<uint32_t>(m.x) & ((1u << (x & 31)) - 1u))) + 1);
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
inline size_t paged_compact_ws(long long N) { return sizeof(int4) * static_cast<size_t>(1 + (N + 31) / 32); }

// Words of shared memory of a compaction.
inline long long paged_compact_words(long long N) { return 2 * ((N + 31) / 32); }

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

// Copies of blocks within a cache: keys, values and their scales. A warp takes 2 KB of a block; bound
// by HBM (every byte read and written once).
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
    if (c.x < 0 && c.y < 0) continue;
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
