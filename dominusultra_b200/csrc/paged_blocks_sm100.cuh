// Blocks of the paged cache (layout in paged_sm100.cuh) that several requests share: forks, copies of
// blocks, and compaction.
//
// fork and compact work on sets of block ids. One cluster of eight CTAs runs a call: each CTA marks the
// ids of its share of the table in bitmaps of its own shared memory (atomics that stay on the SM), then
// takes a slice of the ids, joins that slice of the eight bitmaps over distributed shared memory, and what
// has to be numbered (free blocks, moves) is numbered by counting bits. Cluster barriers stand between
// the phases, so a call is one launch, waits for nothing else and needs no workspace, and since sets and
// counts do not depend on the order of the marks, neither does any result.
#pragma once

#include "du_ptx.cuh"

namespace du {

constexpr int PAGED_SET_CTAS = 8;  // the largest cluster that every device takes
constexpr int PAGED_SET_THREADS = 1024;
constexpr int PAGED_SET_WARPS = PAGED_SET_THREADS / 32;
constexpr int PAGED_SET_SMEM = 200 * 1024;  // bitmaps and per-request words
constexpr int PAGED_SET_PAGES = 128;        // table entries of a row that a warp takes at a time

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
// A word of another CTA's shared memory, at the address that it has in this one's.
__device__ __forceinline__ uint32_t cluster_load(const uint32_t* here, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Sum over the CTA of each thread's x (x[i] >= 0); every thread gets the sum of all, and in `before`
// the sum over the threads below it. `part`: PAGED_SET_WARPS words of shared memory.
__device__ __forceinline__ int block_scan(int x, int* part, int& before) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int in = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += t;
  }
  __syncthreads();  // (part may still be read from the scan before)
  if (lane == 31) part[warp] = in;
  __syncthreads();
  int w = part[lane];  // (one word per warp: PAGED_SET_WARPS is 32)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  const int total = __shfl_sync(0xffffffffu, w, 31);
  const int below = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  before = in - x + (warp > 0 ? below : 0);
  return total;
}
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
  a.kept = !own || s < 0 || s >= p.B;
  if (!a.kept) {
    const int ls = p.lens[s];
    a.kept = ls < 0 || ls > cap || w < 0 || w > ls;
  }
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
// memory; a warp takes 128 entries of a row at a time, and its lanes fetch the lengths of 32 such pieces
// at once. The lowest request is found by comparing the last blocks of those before it, 32 at a time.
//
// Bound by latency: a chain of four loads (source, lengths, entry; ring), five cluster barriers.
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
  const long long pieces = static_cast<long long>(p.B) * per_row;
  const long long all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const long long share = (pieces + all_warps - 1) / all_warps;
  const long long q_first = (static_cast<long long>(rank) * PAGED_SET_WARPS + warp) * share;
  const long long q_end = min(q_first + share, pieces);
  for (long long q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = static_cast<int>(min(32LL, q_end - q0));
    PagedForkAsk a{};
    if (lane < nq) a = paged_fork_ask(p, static_cast<int>((q0 + lane) / per_row));
    for (int i = 0; i < nq; ++i) {
      const int b = static_cast<int>((q0 + i) / per_row);
      const int c0 = static_cast<int>((q0 + i) % per_row) * PAGED_SET_PAGES;
      const int src = __shfl_sync(0xffffffffu, a.src, i);
      const int n = __shfl_sync(0xffffffffu, a.n, i);
      const int pages = __shfl_sync(0xffffffffu, a.pages, i);
      const int old_pages = __shfl_sync(0xffffffffu, a.old_pages, i);
      const bool kept = __shfl_sync(0xffffffffu, static_cast<int>(a.kept), i) != 0;
      const int partly = !kept && n % p.block != 0 ? pages - 1 : -1;
      const int* row_old = p.table + static_cast<long long>(b) * p.width;
      const int* row_new = p.table + static_cast<long long>(src) * p.width;
      int ids[2][PAGED_SET_PAGES / 32];
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        const int page = c0 + 32 * k + lane;
        ids[0][k] = page < old_pages ? row_old[page] : -1;
        ids[1][k] = page < pages ? row_new[page] : -1;
      }
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        const int page = c0 + 32 * k + lane;
        const int x = ids[0][k], y = ids[1][k];
        if (static_cast<unsigned>(x) < static_cast<unsigned>(p.N)) set_bit(before, x);
        if (page < pages) {
          if (static_cast<unsigned>(y) < static_cast<unsigned>(p.N)) {
            set_bit(after, y);
            if (page != partly) set_bit(whole, y);
          } else {
            record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(y));
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
  taken = min(taken, count);
  auto ring_at = [&](long long i) { return static_cast<int>((static_cast<long long>(head) + i) % p.N); };
  if (ring_ok) {
    int at = freed_before;
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      uint32_t m = w < w1 ? before[w] : 0u;
      int lower;
      const int sum = block_scan(__popc(m), part, lower);
      for (int i = at + lower; m; ++i, m &= m - 1u) p.ring[ring_at(static_cast<long long>(count) + i)] = 32 * w + __ffs(static_cast<int>(m)) - 1;
      at += sum;
    }
  }
  if (rank == 0 && tid == 0) {
    p.state_out[0] = ring_ok ? ring_at(taken) : head;
    p.state_out[1] = ring_ok ? count - taken + freed : count;
  }
  // Rows, lengths and pairs.
  for (long long q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = static_cast<int>(min(32LL, q_end - q0));
    int src = 0, entries = 0;    // the row that the request's is copied from, and how much of it
    int own = -1, own_at = -1;   // the block that it gets, and where in the row that goes
    if (lane < nq) {
      const int b = static_cast<int>((q0 + lane) / per_row);
      const PagedForkAsk a = paged_fork_ask(p, b);
      const bool kept = a.kept || !ring_ok;
      int n = kept ? p.lens[b] : a.n, from = -1;
      src = kept ? b : a.src;
      entries = kept ? p.width : a.pages;
      const uint32_t m = needs_all[b >> 5];
      if (!kept && ((m >> (b & 31)) & 1u)) {
        const int r = need_rank[b >> 5] + __popc(m & ((1u << (b & 31)) - 1u));
        if (r < count) {
          own = p.ring[ring_at(r)];
          own_at = a.pages - 1;
          from = last[b];
          if (static_cast<unsigned>(own) >= static_cast<unsigned>(p.N)) record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(own));
        } else {
          entries = a.pages - 1;
          n = entries * p.block;
        }
      }
      if ((q0 + lane) % per_row == 0) {
        p.lens_out[b] = n;
        p.copies[2LL * b] = from;
        p.copies[2LL * b + 1] = own;
      }
    }
    for (int i = 0; i < nq; ++i) {
      const long long b = (q0 + i) / per_row;
      const int c0 = static_cast<int>((q0 + i) % per_row) * PAGED_SET_PAGES;
      const long long from = static_cast<long long>(__shfl_sync(0xffffffffu, src, i)) * p.width;
      const int n = __shfl_sync(0xffffffffu, entries, i);
      const int mine = __shfl_sync(0xffffffffu, own, i), mine_at = __shfl_sync(0xffffffffu, own_at, i);
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        const int page = c0 + 32 * k + lane;
        if (page < p.width) p.table_out[b * p.width + page] = page == mine_at ? mine : (page < n ? p.table[from + page] : -1);
      }
    }
  }
  cluster_sync();  // (no CTA ends while another reads its flags)
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
// the word. The list of moves is written first and serves as the map for the table's entries (a rank in
// the sets, then a load).
//
// Bound by latency, as the fork; five cluster barriers.
__global__ void __cluster_dims__(PAGED_SET_CTAS, 1, 1) __launch_bounds__(PAGED_SET_THREADS, 1)
    paged_compact_kernel(const PagedCompactParams p) {
  extern __shared__ uint32_t sm_set[];
  __shared__ int part[PAGED_SET_WARPS];
  // of this CTA's slice: ids in use, free ids, ids that are both (or none of the cache's); then, from the
  // CTA whose slice holds it: the end t, ids in use from t on and free ids below t in that slice
  __shared__ uint32_t told[6];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int words = (p.N + 31) >> 5;
  const int slice = (words + PAGED_SET_CTAS - 1) / PAGED_SET_CTAS;
  uint32_t* used = sm_set;
  uint32_t* spare = used + words;
  int* rank_of = reinterpret_cast<int*>(spare + words);  // [slice] moves before each word of this slice
  for (int i = tid; i < 2 * words; i += PAGED_SET_THREADS) sm_set[i] = 0u;
  if (tid < 6) told[tid] = 0u;
  griddep_wait();
  const int head = p.state[0], count = p.state[1];
  const bool state_ok = head >= 0 && head < p.N && count >= 0 && count <= p.N;
  __syncthreads();

  const int cap = p.width * p.block;
  const int per_row = (p.width + PAGED_SET_PAGES - 1) / PAGED_SET_PAGES;
  const long long pieces = static_cast<long long>(p.B) * per_row;
  const long long all_warps = PAGED_SET_CTAS * PAGED_SET_WARPS;
  const long long share = (pieces + all_warps - 1) / all_warps;
  const long long q_first = (static_cast<long long>(rank) * PAGED_SET_WARPS + warp) * share;
  const long long q_end = min(q_first + share, pieces);
  // Blocks of a row: -1 for a request whose length is out of range (its row stays as it is).
  auto pages_of = [&](int b) {
    const int n = p.lens[b];
    return n < 0 || n > cap ? -1 : (n + p.block - 1) / p.block;
  };
  for (long long q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = static_cast<int>(min(32LL, q_end - q0));
    int held = 0;
    if (lane < nq) {
      const int b = static_cast<int>((q0 + lane) / per_row);
      held = pages_of(b);
      if (held < 0) record_error(6u, static_cast<unsigned>(b), static_cast<unsigned>(p.lens[b]));
    }
    for (int i = 0; i < nq; ++i) {
      const long long b = (q0 + i) / per_row;
      const int c0 = static_cast<int>((q0 + i) % per_row) * PAGED_SET_PAGES;
      const int n = __shfl_sync(0xffffffffu, held, i);
      int ids[PAGED_SET_PAGES / 32];
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        const int page = c0 + 32 * k + lane;
        ids[k] = page < n ? p.table[b * p.width + page] : 0;
      }
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        if (c0 + 32 * k + lane >= n) continue;
        if (static_cast<unsigned>(ids[k]) < static_cast<unsigned>(p.N)) set_bit(used, ids[k]);
        else record_error(7u, static_cast<unsigned>(b), static_cast<unsigned>(ids[k]));
      }
    }
  }
  const int threads = PAGED_SET_CTAS * PAGED_SET_THREADS;
  const int first = static_cast<int>(rank) * PAGED_SET_THREADS + tid;
  auto ring_at = [&](long long i) { return static_cast<int>((static_cast<long long>(head) + i) % p.N); };
  if (state_ok) {
    for (long long i = first; i < count; i += threads) {
      const int x = p.ring[ring_at(i)];
      if (static_cast<unsigned>(x) < static_cast<unsigned>(p.N)) set_bit(spare, x);
    }
  }
  cluster_sync();

  // This CTA's slice of the ids: the eight CTAs' bits joined and counted.
  const int w0 = min(static_cast<int>(rank) * slice, words), w1 = min(w0 + slice, words);
  int n_used = 0, n_spare = 0, n_both = 0;
  for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) {
    uint32_t u = 0u, f = 0u;
#pragma unroll
    for (uint32_t r = 0; r < PAGED_SET_CTAS; ++r) {
      u |= cluster_load(used + w, r);
      f |= cluster_load(spare + w, r);
    }
    used[w] = u;
    spare[w] = f;
    n_used += __popc(u);
    n_spare += __popc(f);
    n_both += __popc(u & f);
  }
  int below;
  n_used = block_scan(n_used, part, below);
  n_spare = block_scan(n_spare, part, below);
  n_both = block_scan(n_both, part, below);
  if (tid == 0) {
    told[0] = static_cast<uint32_t>(n_used);
    told[1] = static_cast<uint32_t>(n_spare);
    told[2] = static_cast<uint32_t>(n_both);
  }
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
  int end_slice = -1, rest = all_used, before_moves = 0, before_holes = 0, before_left = 0;
#pragma unroll
  for (int r = 0; r < PAGED_SET_CTAS; ++r) {
    if (end_slice < 0) {
      if (rest <= of_used[r] + of_spare[r]) end_slice = r;
      else rest -= of_used[r] + of_spare[r];
    }
  }
  if (static_cast<int>(rank) == end_slice) {
    // (ids of the slice in order: the one before which `rest` of them lie; its word finds it)
    int seen = 0;
    if (rest == 0) {
      if (tid == 0) told[3] = static_cast<uint32_t>(32 * w0);
    } else {
      for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
        const int w = v0 + tid;
        uint32_t m = w < w1 ? used[w] | spare[w] : 0u;
        int at;
        const int c = __popc(m), sum = block_scan(c, part, at);
        int k = rest - seen - at;  // the k-th bit of this word is the last of the lowest
        if (k >= 1 && k <= c) {
          for (; k > 1; --k) m &= m - 1u;
          told[3] = static_cast<uint32_t>(32 * w + __ffs(static_cast<int>(m)));
        }
        seen += sum;
      }
    }
    __syncthreads();
    const int end = static_cast<int>(told[3]);
    int moves = 0, holes = 0;
    for (int w = w0 + tid; w < w1; w += PAGED_SET_THREADS) {
      const int d = end - 32 * w;
      const uint32_t low = d <= 0 ? 0u : (d >= 32 ? 0xffffffffu : (1u << d) - 1u);
      moves += __popc(used[w] & ~low);
      holes += __popc(spare[w] & low);
    }
    moves = block_scan(moves, part, below);
    holes = block_scan(holes, part, below);
    if (tid == 0) {
      told[4] = static_cast<uint32_t>(moves);
      told[5] = static_cast<uint32_t>(holes);
    }
  }
  cluster_sync();
  const int end = static_cast<int>(cluster_load(told + 3, static_cast<uint32_t>(end_slice)));
  const int end_moves = static_cast<int>(cluster_load(told + 4, static_cast<uint32_t>(end_slice)));
  const int end_holes = static_cast<int>(cluster_load(told + 5, static_cast<uint32_t>(end_slice)));
  int all_moves = end_moves;
#pragma unroll
  for (int r = 0; r < PAGED_SET_CTAS; ++r) {
    if (r > end_slice) all_moves += of_used[r];
    if (r >= static_cast<int>(rank)) continue;
    before_moves += r == end_slice ? end_moves : (r > end_slice ? of_used[r] : 0);
    before_holes += r == end_slice ? end_holes : (r < end_slice ? of_spare[r] : 0);
    before_left += r == end_slice ? of_used[r] + of_spare[r] - rest : (r > end_slice ? of_used[r] + of_spare[r] : 0);
  }
  if (ok) {
    for (int v0 = w0; v0 < w1; v0 += PAGED_SET_THREADS) {
      const int w = v0 + tid;
      const int d = end - 32 * w;
      const uint32_t low = d <= 0 ? 0u : (d >= 32 ? 0xffffffffu : (1u << d) - 1u);
      const uint32_t u = w < w1 ? used[w] : 0u, f = w < w1 ? spare[w] : 0u;
      uint32_t move = u & ~low, hole = f & low, left = (u | f) & ~low;
      int at_move, at_hole, at_left;
      const int s_move = block_scan(__popc(move), part, at_move);
      const int s_hole = block_scan(__popc(hole), part, at_hole);
      const int s_left = block_scan(__popc(left), part, at_left);
      if (w < w1) {
        used[w] = move;
        rank_of[w - w0] = before_moves + at_move;
      }
      for (int i = before_moves + at_move; move; ++i, move &= move - 1u) p.copies[2LL * i] = 32 * w + __ffs(static_cast<int>(move)) - 1;
      for (int i = before_holes + at_hole; hole; ++i, hole &= hole - 1u) p.copies[2LL * i + 1] = 32 * w + __ffs(static_cast<int>(hole)) - 1;
      for (int i = before_left + at_left; left; ++i, left &= left - 1u) p.ring_out[i] = 32 * w + __ffs(static_cast<int>(left)) - 1;
      before_moves += s_move;
      before_holes += s_hole;
      before_left += s_left;
    }
  } else {
    all_moves = 0;
  }
  for (long long i = 2LL * all_moves + first; i < 2LL * (p.N / 2); i += threads) p.copies[i] = -1;
  for (long long i = (ok ? count : 0) + first; i < p.N; i += threads) p.ring_out[i] = ok ? -1 : p.ring[i];
  if (rank == 0 && tid == 0) {
    p.state_out[0] = ok ? 0 : head;
    p.state_out[1] = count;
  }
  cluster_sync();

  for (long long q0 = q_first; q0 < q_end; q0 += 32) {
    const int nq = static_cast<int>(min(32LL, q_end - q0));
    const int held = lane < nq ? pages_of(static_cast<int>((q0 + lane) / per_row)) : 0;
    for (int i = 0; i < nq; ++i) {
      const long long b = (q0 + i) / per_row;
      const int c0 = static_cast<int>((q0 + i) % per_row) * PAGED_SET_PAGES;
      const int n = __shfl_sync(0xffffffffu, held, i);
      const bool whole_row = !ok || n < 0;
#pragma unroll
      for (int k = 0; k < PAGED_SET_PAGES / 32; ++k) {
        const int page = c0 + 32 * k + lane;
        if (page >= p.width) continue;
        int x = whole_row || page < n ? p.table[b * p.width + page] : -1;
        if (!whole_row && x >= end && x < p.N) {
          const int w = x >> 5, s = w / slice;
          const uint32_t m = cluster_load(used + w, static_cast<uint32_t>(s)) & ((1u << (x & 31)) - 1u);
          const int r = static_cast<int>(cluster_load(reinterpret_cast<uint32_t*>(rank_of + (w - s * slice)), static_cast<uint32_t>(s))) + __popc(m);
          x = __ldcg(p.copies + 2LL * r + 1);
        }
        p.table_out[b * p.width + page] = x;
      }
    }
  }
  cluster_sync();  // (no CTA ends while another reads its sets)
}

// Words of shared memory of a compaction.
inline long long paged_compact_words(long long N) {
  const long long words = (N + 31) / 32;
  return 2 * words + (words + PAGED_SET_CTAS - 1) / PAGED_SET_CTAS;
}

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
