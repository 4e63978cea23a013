// The pages of a paged cache: which sequences list them, and where they lie.  Sequences fork (q40_page_fork), get pages for their next tokens or give some back
// (q40_page_extend), and pages in use move to the front of their pools (q40_page_compact), by what the device's books say: a table of page ids and a length for
// each sequence, and for each page how many sequences list it (0: it is free).  Nothing goes by way of the host, so that a captured step can be replayed.
//
// Free pages are handed out in ascending order, to the sequences in theirs: results do not depend on which thread comes first.
//
// Few sequences and pages: one launch.  Every CTA makes the whole plan for itself, in shared memory, from books of some ten thousand numbers that lie in L2, and then
// writes its share of the tables and moves its share of what the pools hold, so that no CTA waits for another.  Books that are written in place are another matter: one
// cluster of eight CTAs, which have all read before one writes.
// Many: a plan by one cluster (each warp has a run of pages, which it counts through by ballots; CTAs hand each other their sums through distributed shared memory;
// a page that is the r-th free one looks up the sequence that wants it in the sums of what they want), and a second launch, of all SMs, for tables and pools.
//
// What bounds it: few sequences, a chain of loads (lengths, the table, references) and two scans; pools that move, HBM.
#include <cooperative_groups.h>

#include <algorithm>

#include "pages_common.cuh"

namespace q40 {
namespace books {

namespace cg = cooperative_groups;

constexpr int CLUSTER = 8, NT = 1024, WARPS = NT / 32;      // of a plan
constexpr int MOST_SEQUENCES = 16384;                       // of an extension: what they want is summed in shared memory
constexpr int CHUNK = 1024, ROW_THREADS = 256;              // entries of a table that a block takes at a time
constexpr int FEW_ROWS = NT, FEW_PAGES = 16384;             // of calls whose plan each CTA makes for itself
constexpr int FEW_LOADS = 4, MANY_LOADS = 8;                // of 512 bytes, that a warp has under way when it moves a page
constexpr int UNIT = 128;                                   // entries of a table that a warp takes at a time
constexpr int FORK_UNITS = 2;                               // ... and how many of these it holds at once

struct Books {
  const int32_t *table, *lens, *refs;
  int64_t ld, ld_out;
  int32_t *table_out, *lens_out, *refs_out;
  int B, W, pages, page_size, page_shift;
  __device__ __forceinline__ int pages_of(int tokens) const {        // tokens >= 0
    return (int)(page_shift >= 0 ? ((unsigned)tokens + (unsigned)page_size - 1u) >> page_shift : ((unsigned)tokens + (unsigned)page_size - 1u) / (unsigned)page_size);
  }
  // A length that the table has room for
  __device__ __forceinline__ int length(int b) const { return (int)min((int64_t)max(lens[b], 0), (int64_t)W * page_size); }
  __device__ __forceinline__ bool valid(int id) const { return (unsigned)id < (unsigned)pages; }
};

struct Pools {
  unsigned char *k, *v;              // [heads, P, row_bytes]
  float *ks, *vs;                    // [heads, P / page_size], or nullptr
  int heads, row_bytes;
  int64_t P, scale_stride;
};

// Pages that move: the first rows[i] rows of page src[i] (nullptr: all) to page dst[i]
struct Moves {
  int *n, *src, *dst, *rows;
};

// What moves, by warps, this one at `at` of `step`: the first rows[i] rows (nullptr: all) of n pages src[i] to dst[i], of each head, keys or values, a piece of LOADS x 512 bytes at a time
template <int LOADS>
__device__ __forceinline__ void move(const Pools& pools, int page_size, const int* src_of, const int* dst_of, const int* rows, int n, int64_t at, int64_t step) {
  constexpr int PIECE = LOADS * 512;
  const int lane = threadIdx.x & 31;
  const int pieces = (int)(((int64_t)page_size * pools.row_bytes + PIECE - 1) / PIECE);
  const int64_t per = (int64_t)2 * pools.heads * pieces;
  if (per == 0) return;
  int64_t i = at / per, rest = at % per;
  const int64_t i_step = step / per, rest_step = step % per;
  while (i < n) {
    const int src = src_of[i], dst = dst_of[i], piece = (int)(rest % pieces);
    const int64_t bytes = (int64_t)(rows ? rows[i] : page_size) * pools.row_bytes;
    int head = (int)(rest / pieces);
    const bool values = head >= pools.heads;
    if (values) head -= pools.heads;
    unsigned char* const pool = (values ? pools.v : pools.k) + (int64_t)head * pools.P * pools.row_bytes;
    const unsigned char* const from = pool + (int64_t)src * page_size * pools.row_bytes;
    unsigned char* const to = pool + (int64_t)dst * page_size * pools.row_bytes;
    uint4 x[LOADS];
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const int64_t off = (int64_t)piece * PIECE + c * 512 + lane * 16;
      if (off < bytes) x[c] = *reinterpret_cast<const uint4*>(from + off);
    }
    if (piece == 0 && lane == 0 && pools.ks) {
      float* const scale = (values ? pools.vs : pools.ks) + (int64_t)head * pools.scale_stride;
      scale[dst] = scale[src];
    }
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const int64_t off = (int64_t)piece * PIECE + c * 512 + lane * 16;
      if (off < bytes) *reinterpret_cast<uint4*>(to + off) = x[c];
    }
    i += i_step;
    rest += rest_step;
    if (rest >= per) {
      rest -= per;
      ++i;
    }
  }
}

// ---- forks ---------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
fork_refs_kernel(const int32_t* refs, int32_t* out, int n) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) out[i] = refs[i];
}

// A sequence lists page `now` where it listed `old` (-1: none)
__device__ __forceinline__ void count(const Books& b, int now, int old) {
  if (now == old) return;
  if (b.valid(now)) atomicAdd(b.refs_out + now, 1);
  if (b.valid(old)) atomicAdd(b.refs_out + old, -1);
}

__global__ void __launch_bounds__(ROW_THREADS)
fork_rows_kernel(const Books b, const int32_t* parents, int chunks) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x / chunks, j0 = (blockIdx.x % chunks) * CHUNK + threadIdx.x;
  const int p = parents[row];
  const bool there = (unsigned)p < (unsigned)b.B;
  const int len = there ? b.length(p) : 0, n_new = b.pages_of(len), n_old = b.pages_of(b.length(row));
  const int32_t* const from = b.table + (int64_t)(there ? p : 0) * b.ld;
  const int32_t* const own = b.table + (int64_t)row * b.ld;
  int32_t* const out = b.table_out + (int64_t)row * b.ld_out;
  if (j0 == 0) b.lens_out[row] = len;
#pragma unroll
  for (int i = 0; i < CHUNK / ROW_THREADS; ++i) {
    const int j = j0 + i * ROW_THREADS;
    if (j >= b.W) break;
    const int id = j < n_new ? from[j] : -1;
    out[j] = max(id, 0);
    if (p == row) continue;
    count(b, id, j < n_old ? own[j] : -1);
  }
}

// Few: one cluster, whose warps have all read what they write, units of a row's entries, before one of them does
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(NT)
fork_few_kernel(const Books b, const int32_t* parents, int units, int row_units) {
  const int lane = threadIdx.x & 31, warp = (int)blockIdx.x * WARPS + (int)(threadIdx.x >> 5);
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int now[FORK_UNITS][4], old[FORK_UNITS][4], len[FORK_UNITS];       // page ids, -1: none
  bool changes[FORK_UNITS];
#pragma unroll
  for (int u = 0; u < FORK_UNITS; ++u) {
    const int unit = warp + u * CLUSTER * WARPS;
    if (unit >= units) break;
    const int row = unit / row_units, j0 = unit % row_units * UNIT + lane, p = parents[row];
    const bool there = (unsigned)p < (unsigned)b.B;
    len[u] = there ? b.length(p) : 0;
    changes[u] = p != row;
    const int n_new = b.pages_of(len[u]), n_old = b.pages_of(b.length(row));
#pragma unroll
    for (int i = 0; i < UNIT / 32; ++i) {
      const int j = j0 + 32 * i;
      now[u][i] = j < n_new ? b.table[(int64_t)p * b.ld + j] : -1;
      old[u][i] = j < n_old ? b.table[(int64_t)row * b.ld + j] : -1;
    }
  }
  if (b.refs_out != b.refs)
    for (int i = blockIdx.x * NT + threadIdx.x; i < b.pages; i += CLUSTER * NT) b.refs_out[i] = b.refs[i];
  cg::this_cluster().sync();
#pragma unroll
  for (int u = 0; u < FORK_UNITS; ++u) {
    const int unit = warp + u * CLUSTER * WARPS;
    if (unit >= units) break;
    const int row = unit / row_units, j0 = unit % row_units * UNIT + lane;
    int32_t* const out = b.table_out + (int64_t)row * b.ld_out;
    if (j0 == 0) b.lens_out[row] = len[u];
#pragma unroll
    for (int i = 0; i < UNIT / 32; ++i) {
      if (j0 + 32 * i >= b.W) break;
      out[j0 + 32 * i] = max(now[u][i], 0);
      if (changes[u]) count(b, now[u][i], old[u][i]);
    }
  }
}

// ---- what plans share ----------------------------------------------------------------------------------------------
// A warp's run of pages, in order over the cluster
struct Run {
  int lo, hi;
  // that of warp `w` of `warps`
  __device__ __forceinline__ Run(int pages, int w, int warps) {
    const int each = ((pages + warps - 1) / warps + 31) / 32 * 32;
    const int64_t first = (int64_t)w * each;
    lo = (int)min(first, (int64_t)pages);
    hi = (int)min(first + each, (int64_t)pages);
  }
};
// The pages of a run, 32 at a time, four of these requested together, the first before what they are for: f(first page, this lane's references; 0 behind the end)
struct Ahead {
  int r[4];
  __device__ __forceinline__ Ahead(const int32_t* refs, const Run& run, int p0) {
    const int p = p0 + (int)(threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = p + 32 * i < run.hi ? refs[p + 32 * i] : 0;
  }
};
template <class F>
__device__ __forceinline__ void through(const int32_t* refs, const Run& run, Ahead ahead, F f) {
  for (int p0 = run.lo; p0 < run.hi; p0 += 128) {
    if (p0 > run.lo) ahead = Ahead(refs, run, p0);
    const int(&r)[4] = ahead.r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + 32 * i < run.hi) f(p0 + 32 * i, r[i]);
  }
}
template <class F>
__device__ __forceinline__ void through(const int32_t* refs, const Run& run, F f) { through(refs, run, Ahead(refs, run, run.lo), f); }
// Sum of x over the warps in front of this one, and over all of the CTA (each lane of a warp has its x).  All threads call it
__device__ __forceinline__ int before_in_cta(int x, int* sums, int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) sums[warp] = x;
  __syncthreads();
  int mine = sums[lane], front = lane < warp ? mine : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mine += __shfl_xor_sync(0xffffffffu, mine, o);
    front += __shfl_xor_sync(0xffffffffu, front, o);
  }
  all = mine;
  return front;
}

// ---- extension -----------------------------------------------------------------------------------------------------
// (what the kernels with less to tell get: with 216 bytes of arguments instead of 160 a launch takes 0.5 us longer)
struct Additions : Books {
  const int32_t* add;
};
struct Extension : Additions {
  int *writers, *last;               // of each page: sequences that write to it behind its rows, and the last of them
  int4* plan;                        // of each sequence: entries that stay, entries in all, entries before, length
  Moves moves;
};

struct Growth {
  __device__ __forceinline__ Growth() : n(0), m(0), n0(0), n1(0), tail(-1), shared(0), grows(false) {}
  int n, m, n0, n1;                  // tokens and pages, before and after
  int tail, shared;                  // a page that is in part filled and will be written to (-1: none), and its references
  bool grows;                        // into pages that the table has room for
  __device__ __forceinline__ Growth(const Additions& a, int b) {
    n = a.length(b);
    const int add = a.add[b];
    const int64_t to = max((int64_t)n + add, (int64_t)0);
    m = (int)min(to, (int64_t)0x7fffffff);
    n0 = a.pages_of(n);
    n1 = a.pages_of(m);
    grows = add > 0 && to <= 0x7fffffff && n1 <= a.W;
    tail = -1;
    shared = 0;
    if (grows && n % a.page_size != 0) {
      const int id = a.table[(int64_t)b * a.ld + n0 - 1];
      if (a.valid(id)) {
        tail = id;
        shared = a.refs[id];
      } else {
        grows = false;
      }
    }
  }
};

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(NT)
extend_plan_kernel(const Extension a) {
  constexpr int COPIES = 1 << 31, GROWS = 1 << 30, WANTS = 1 << 29, PAGES = WANTS - 1;
  extern __shared__ int wanted[];                // [B + 1] pages that the sequences in front want, at most `pages` + 1
  int* const info = wanted + a.B + 1;            // [B] PAGES: how many before; GROWS, WANTS any page or keeps one that others copy, COPIES one
  __shared__ int sums[WARPS], s_free;
  __shared__ long long s_sums[WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Pages that several sequences list and some will write to
  for (int b = rank * NT + tid; b < a.B; b += CLUSTER * NT) {
    const Growth g(a, b);
    if (g.tail >= 0 && g.shared > 1) {
      a.writers[g.tail] = 0;
      a.last[g.tail] = -1;
    }
  }
  if (rank == 0 && tid == 0) *a.moves.n = 0;
  const Run run(a.pages, rank * WARPS + (tid >> 5), CLUSTER * WARPS);
  int free = 0;
  through(a.refs, run, [&](int p0, int r) {
    const int p = p0 + lane;
    free += __popc(__ballot_sync(0xffffffffu, p < run.hi && r <= 0));
    if (a.refs_out != a.refs && p < run.hi) a.refs_out[p] = r;
  });
  int in_cta;
  int rank_of_free = before_in_cta(free, sums, in_cta);
  if (tid == 0) s_free = in_cta;
  cluster.sync();
  for (int b = rank * NT + tid; b < a.B; b += CLUSTER * NT) {
    const Growth g(a, b);
    if (g.tail >= 0 && g.shared > 1) {
      atomicAdd(a.writers + g.tail, 1);
      atomicMax(a.last + g.tail, b);
    }
  }
  int all_free = 0;
  for (int i = 0; i < CLUSTER; ++i) {
    const int x = *cluster.map_shared_rank(&s_free, i);
    if (i < rank) rank_of_free += x;
    all_free += x;
  }
  cluster.sync();

  // What each sequence wants; every CTA for itself
  long long carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += NT) {
    const int b = b0 + tid;
    int need = 0;
    if (b < a.B) {
      const Growth g(a, b);
      bool copies = false, keeps = false;
      if (g.grows) {
        // Of sequences that all write to a page which no other lists, the last keeps it.  One of the others that gets no copy lists it still: the last is refused with it
        const bool shares = g.tail >= 0 && g.shared > 1;
        keeps = shares && __ldcg(a.writers + g.tail) == g.shared && __ldcg(a.last + g.tail) == b;
        copies = shares && !keeps;
        need = g.n1 - g.n0 + (copies ? 1 : 0);
      }
      info[b] = g.n0 | (g.grows ? GROWS : 0) | (need || keeps ? WANTS : 0) | (copies ? COPIES : 0);
    }
    long long x = need;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_sums[warp] = x;
    __syncthreads();
    long long front = 0, all = 0;
    for (int w = 0; w < WARPS; ++w) {
      const long long y = s_sums[w];
      if (w < warp) front += y;
      all += y;
    }
    if (b < a.B) wanted[b] = (int)min(carry + front + x - need, (long long)a.pages + 1);
    carry += all;
  }
  if (tid == 0) wanted[a.B] = (int)min(carry, (long long)a.pages + 1);
  cluster.sync();                                // the books are read; what is written may be they

  // Once a sequence does not get what it wants, none behind it gets any
  const int given = min(wanted[a.B], all_free);
  if (rank_of_free < given)
    through(a.refs, run, [&](int p0, int r) {
      const int p = p0 + lane;
      const bool is_free = p < run.hi && r <= 0;
      const uint32_t mask = __ballot_sync(0xffffffffu, is_free);
      const int at = rank_of_free + __popc(mask & ((1u << lane) - 1u));
      rank_of_free += __popc(mask);
      if (!is_free || at >= given) return;
      int b = 0, above = a.B;                    // the last that begins at `at` or in front of it
      while (above - b > 1) {
        const int mid = (b + above) >> 1;
        if (wanted[mid] <= at) b = mid;
        else above = mid;
      }
      if (wanted[b + 1] > all_free) return;
      const bool copies = info[b] & COPIES;
      const int n0 = info[b] & PAGES, j = n0 - (copies ? 1 : 0) + at - wanted[b];
      int32_t* const entry = a.table_out + (int64_t)b * a.ld_out + j;
      if (copies && at == wanted[b]) {
        const int i = atomicAdd(a.moves.n, 1);
        a.moves.src[i] = a.table[(int64_t)b * a.ld + j];
        a.moves.dst[i] = p;
        a.moves.rows[i] = a.length(b) % a.page_size;
      }
      *entry = p;
      a.refs_out[p] = 1;
    });
  for (int b = rank * NT + tid; b < a.B; b += CLUSTER * NT) {
    const int n = a.length(b), add = a.add[b], n0 = info[b] & PAGES;
    int4 plan = make_int4(n0, n0, n0, n);
    if (add <= 0) {
      const int m = (int)max((int64_t)n + add, (int64_t)0), n1 = a.pages_of(m);
      plan = make_int4(n1, n1, n0, m);
    } else if ((info[b] & GROWS) && (!(info[b] & WANTS) || wanted[b + 1] <= all_free)) {
      plan = make_int4(n0 - (info[b] & COPIES ? 1 : 0), a.pages_of(n + add), n0, n + add);
    }
    a.plan[b] = plan;
  }
}

// Few: every CTA plans for itself.  A thread has a sequence
template <bool IN_PLACE>
__global__ void __launch_bounds__(NT)
extend_few_kernel(const Additions a, const Pools pools) {
  extern __shared__ int4 few_smem[];
  int* const tails = reinterpret_cast<int*>(few_smem);       // [FEW_ROWS] pages that several list and this one writes to, or -1
  int* const first = tails + FEW_ROWS;           // [FEW_ROWS] rank of the first page that it gets
  int* const keep = first + FEW_ROWS;            // [FEW_ROWS] entries that stay
  int* const end = keep + FEW_ROWS;              // [FEW_ROWS] entries in all
  int* const before = end + FEW_ROWS;            // [FEW_ROWS] entries before
  int* const src = before + FEW_ROWS;            // [FEW_ROWS] pages that are copied, ..
  int* const dst = src + FEW_ROWS;
  int* const rows = dst + FEW_ROWS;
  int* const handed = rows + FEW_ROWS;           // [pages] free ones, in order
  int* const refs = handed + (a.pages + 3) / 4 * 4;          // [pages], of the CTA that counts
  __shared__ int sums[WARPS], masks[FEW_PAGES / 32];               // (masks: a bit for each free page)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const Run run(a.pages, warp, WARPS);
  const Ahead ahead(a.refs, run, run.lo);
  const bool there = tid < a.B;
  Growth g;
  if (there) g = Growth(a, tid);
  int free = 0;
  through(a.refs, run, ahead, [&](int p0, int r) {
    const uint32_t mask = __ballot_sync(0xffffffffu, p0 + lane < run.hi && r <= 0);
    free += __popc(mask);
    if (lane == 0) masks[p0 / 32] = (int)mask;
    if (!IN_PLACE && cta == 0 && p0 + lane < run.hi) refs[p0 + lane] = r;
  });
  const bool shares = there && g.tail >= 0 && g.shared > 1;
  tails[tid] = shares ? g.tail : -1;
  int all_free;
  int rank = before_in_cta(free, sums, all_free);
  bool copies = shares;
  if (shares) {                                  // of sequences that all write to a page which no other lists, the last keeps it (see extend_plan_kernel)
    int writers = 0, last = 0;
    for (int b = 0; b < a.B; b += 4) {
      const int4 t = reinterpret_cast<const int4*>(tails)[b / 4];
      const bool same[4] = {t.x == g.tail, t.y == g.tail, t.z == g.tail, t.w == g.tail};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (same[i]) {
          ++writers;
          last = b + i;
        }
    }
    copies = !(writers == g.shared && last == tid);
  }
  const int need = g.grows ? min(g.n1 - g.n0 + (copies ? 1 : 0), a.pages + 1) : 0;       // (their sum is below 2^25)
  int upto = need, wanted, n_moves;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  upto += before_in_cta(__shfl_sync(0xffffffffu, upto, 31), sums, wanted);
  const bool granted = g.grows && ((need == 0 && copies == shares) || upto <= all_free);
  const bool moves = granted && copies;
  const uint32_t moving = __ballot_sync(0xffffffffu, moves);
  const int front = before_in_cta(__popc(moving), sums, n_moves) + __popc(moving & ((1u << lane) - 1u));       // (each CTA has the same order)
  for (int p0 = run.lo; p0 < run.hi; p0 += 32) {
    const uint32_t mask = (uint32_t)masks[p0 / 32];
    if ((mask >> lane) & 1u) handed[rank + __popc(mask & ((1u << lane) - 1u))] = p0 + lane;
    rank += __popc(mask);
  }
  int len = g.n;
  if (there) {
    const bool gives = a.add[tid] <= 0;
    if (gives || granted) len = g.m;
    first[tid] = upto - need;
    keep[tid] = granted ? g.n0 - (copies ? 1 : 0) : gives ? g.n1 : g.n0;
    end[tid] = gives || granted ? g.n1 : g.n0;
    before[tid] = g.n0;
  }
  __syncthreads();
  if (moves) {
    src[front] = g.tail;
    dst[front] = handed[upto - need];
    rows[front] = g.n % a.page_size;
  }
  if (IN_PLACE) cg::this_cluster().sync();
  else __syncthreads();

  if (there && cta == 0) a.lens_out[tid] = len;
  const int units = (a.W + UNIT - 1) / UNIT;
  for (int64_t u = (int64_t)cta * WARPS + warp; u < (int64_t)a.B * units; u += (int64_t)ctas * WARPS) {
    const int b = (int)(u / units), j0 = (int)(u % units) * UNIT + lane, stay = keep[b], stop = end[b], was = before[b];
    const int32_t* const from = a.table + (int64_t)b * a.ld;
    int32_t* const out = a.table_out + (int64_t)b * a.ld_out;
#pragma unroll
    for (int i = 0; i < UNIT / 32; ++i) {
      const int j = j0 + 32 * i;
      if (j >= a.W) break;
      if (j < stay) {
        if (!IN_PLACE) out[j] = from[j];
      } else if (j < stop) {
        const int page = handed[first[b] + j - stay];
        out[j] = page;
        if (IN_PLACE) a.refs_out[page] = 1;
      } else {
        if (IN_PLACE && j < was && a.valid(from[j])) atomicAdd(a.refs_out + from[j], -1);
        out[j] = 0;
      }
    }
  }
  if (IN_PLACE) {
    if (moves && cta == 0) atomicAdd(a.refs_out + g.tail, -1);
  } else if (cta == 0) {
    if (moves) atomicAdd(refs + g.tail, -1);
    for (int b = warp; b < a.B; b += WARPS) {
      for (int j = keep[b] + lane; j < end[b]; j += 32) refs[handed[first[b] + j - keep[b]]] = 1;
      for (int j = end[b] + lane; j < before[b]; j += 32) {
        const int id = a.table[(int64_t)b * a.ld + j];
        if (a.valid(id)) atomicAdd(refs + id, -1);
      }
    }
    __syncthreads();
    for (int p = tid; p < a.pages; p += NT) a.refs_out[p] = refs[p];
  }
  // (the CTA that counts comes last)
  move<FEW_LOADS>(pools, a.page_size, src, dst, rows, n_moves, (int64_t)(ctas - 1 - cta) * WARPS + warp, (int64_t)ctas * WARPS);
}

// ---- compaction ----------------------------------------------------------------------------------------------------
struct Moving : Books {
  int32_t* where;                    // [pages] a page's new id, or -1 (free)
};
struct Compaction : Moving {
  int* old_refs;                     // of the pages that move
  Moves moves;
};

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(NT)
compact_plan_kernel(const Compaction a) {
  __shared__ int sums[WARPS], s_used, s_movers, s_holes;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Run run(a.pages, rank * WARPS + (tid >> 5), CLUSTER * WARPS);
  int used = 0, all;
  through(a.refs, run, [&](int p0, int r) { used += __popc(__ballot_sync(0xffffffffu, p0 + lane < run.hi && r > 0)); });
  before_in_cta(used, sums, all);
  if (tid == 0) s_used = all;
  cluster.sync();
  int end = 0;                                   // of the front: as many pages as are in use
  for (int i = 0; i < CLUSTER; ++i) end += *cluster.map_shared_rank(&s_used, i);
  int movers = 0, holes = 0;
  if (run.hi <= end) holes = run.hi - run.lo - used;
  else if (run.lo >= end) movers = used;
  else
    through(a.refs, run, [&](int p0, int r) {
      const int p = p0 + lane;
      movers += __popc(__ballot_sync(0xffffffffu, p < run.hi && p >= end && r > 0));
      holes += __popc(__ballot_sync(0xffffffffu, p < run.hi && p < end && r <= 0));
    });
  int mover = before_in_cta(movers, sums, all);
  if (tid == 0) s_movers = all;
  int hole = before_in_cta(holes, sums, all);
  if (tid == 0) s_holes = all;
  cluster.sync();
  int n = 0;
  for (int i = 0; i < CLUSTER; ++i) {
    const int x = *cluster.map_shared_rank(&s_movers, i);
    n += x;
    if (i < rank) {
      mover += x;
      hole += *cluster.map_shared_rank(&s_holes, i);
    }
  }
  through(a.refs, run, [&](int p0, int r) {
    const int p = p0 + lane;
    const bool there = p < run.hi, in_use = there && r > 0, front = p < end;
    const uint32_t moves = __ballot_sync(0xffffffffu, in_use && !front), free = __ballot_sync(0xffffffffu, there && front && !in_use);
    const uint32_t below = (1u << lane) - 1u;
    if (in_use && !front) {
      const int i = mover + __popc(moves & below);
      a.moves.src[i] = p;
      a.old_refs[i] = r;
    } else if (there) {
      a.where[p] = in_use ? p : -1;
    }
    if (there && front && !in_use) a.moves.dst[hole + __popc(free & below)] = p;
    else if (there) a.refs_out[p] = front ? r : 0;
    mover += __popc(moves);
    hole += __popc(free);
  });
  if (rank == 0 && tid == 0) *a.moves.n = n;
  cluster.sync();
  for (int i = rank * NT + tid; i < n; i += CLUSTER * NT) {
    const int dst = __ldcg(a.moves.dst + i);
    a.where[__ldcg(a.moves.src + i)] = dst;
    a.refs_out[dst] = __ldcg(a.old_refs + i);
  }
}

// Few: every CTA plans for itself
template <bool IN_PLACE>
__global__ void __launch_bounds__(NT)
compact_few_kernel(const Moving a, const Pools pools) {
  extern __shared__ int4 few_smem[];
  int* const used = reinterpret_cast<int*>(few_smem);        // [FEW_PAGES / 32] a bit for each page in use
  int* const counted = used + FEW_PAGES / 32;    // [FEW_PAGES / 32] pages in use in front of these 32
  int* const src = counted + FEW_PAGES / 32;     // [pages / 2 + 1] pages that move
  int* const dst = src + a.pages / 2 + 1;        // [pages / 2 + 1] free ones in front
  __shared__ int sums[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Run run(a.pages, warp, WARPS);
  through(a.refs, run, [&](int p0, int r) {
    const uint32_t mask = __ballot_sync(0xffffffffu, p0 + lane < run.hi && r > 0);
    if (lane == 0) used[p0 / 32] = (int)mask;
  });
  __syncthreads();
  const int words = (a.pages + 31) / 32;         // a thread has one
  const uint32_t mine = tid < words ? (uint32_t)used[tid] : 0u;
  int upto = __popc(mine), n_used;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  upto += before_in_cta(__shfl_sync(0xffffffffu, upto, 31), sums, n_used);
  if (tid < words) counted[tid] = upto - __popc(mine);
  __syncthreads();
  const auto in_front = [&](int p) { return p < a.pages ? counted[p / 32] + __popc((uint32_t)used[p / 32] & ((1u << (p & 31)) - 1u)) : n_used; };
  const auto in_use = [&](int p) { return ((uint32_t)used[p / 32] >> (p & 31)) & 1u; };
  const int staying = in_front(n_used), n_moves = n_used - staying;       // pages in use among the first n_used
  for (int p = tid; p < a.pages; p += NT) {
    if (p >= n_used && in_use(p)) src[in_front(p) - staying] = p;
    if (p < n_used && !in_use(p)) dst[p - in_front(p)] = p;
  }
  __syncthreads();
  const auto goes_to = [&](int p) { return !in_use(p) ? -1 : p < n_used ? p : dst[in_front(p) - staying]; };
  // What a page of the front has in references: its own, or those of the page that comes
  constexpr int EACH = IN_PLACE ? FEW_PAGES / (CLUSTER * NT) : 1;
  int r[EACH];
  const auto refs_of = [&](int p) { return p >= n_used ? 0 : a.refs[in_use(p) ? p : src[p - in_front(p)]]; };
  if (IN_PLACE) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int p = (i * CLUSTER + cta) * NT + tid;
      r[i] = p < a.pages ? refs_of(p) : 0;
    }
    cg::this_cluster().sync();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int p = (i * CLUSTER + cta) * NT + tid;
      if (p < a.pages) a.refs_out[p] = r[i];
    }
  }
  for (int p = cta * NT + tid; p < a.pages; p += ctas * NT) {
    a.where[p] = goes_to(p);
    if (!IN_PLACE) a.refs_out[p] = refs_of(p);
  }
  const int units = (a.W + UNIT - 1) / UNIT;
  for (int64_t u = (int64_t)cta * WARPS + warp; u < (int64_t)a.B * units; u += (int64_t)ctas * WARPS) {
    const int b = (int)(u / units), j0 = (int)(u % units) * UNIT + lane, n = a.pages_of(a.length(b));
    const int32_t* const from = a.table + (int64_t)b * a.ld;
    int32_t* const out = a.table_out + (int64_t)b * a.ld_out;
#pragma unroll
    for (int i = 0; i < UNIT / 32; ++i) {
      const int j = j0 + 32 * i;
      if (j >= a.W) break;
      int id = j < n ? from[j] : 0;
      if (j < n && a.valid(id)) id = max(goes_to(id), 0);
      out[j] = id;
    }
  }
  move<FEW_LOADS>(pools, a.page_size, src, dst, nullptr, n_moves, (int64_t)cta * WARPS + warp, (int64_t)ctas * WARPS);
}

// ---- tables and pools ----------------------------------------------------------------------------------------------
__device__ __forceinline__ void table_chunk(const Extension& a, int b, int j0) {
  const int4 plan = a.plan[b];
  const int32_t* const from = a.table + (int64_t)b * a.ld;
  int32_t* const out = a.table_out + (int64_t)b * a.ld_out;
  const bool in_place = a.table == a.table_out;
  if (j0 == 0) a.lens_out[b] = plan.w;
#pragma unroll
  for (int i = 0; i < CHUNK / ROW_THREADS; ++i) {
    const int j = j0 + i * ROW_THREADS;
    if (j >= a.W) break;
    if (j < plan.x) {
      if (!in_place) out[j] = from[j];
    } else if (j >= plan.y) {
      if (j < plan.z && a.valid(from[j])) atomicAdd(a.refs_out + from[j], -1);
      out[j] = 0;
    }
  }
}
__device__ __forceinline__ void table_chunk(const Compaction& a, int b, int j0) {
  const int n = a.pages_of(a.length(b));
  const int32_t* const from = a.table + (int64_t)b * a.ld;
  int32_t* const out = a.table_out + (int64_t)b * a.ld_out;
#pragma unroll
  for (int i = 0; i < CHUNK / ROW_THREADS; ++i) {
    const int j = j0 + i * ROW_THREADS;
    if (j >= a.W) break;
    int id = j < n ? from[j] : 0;
    if (j < n && a.valid(id)) id = max(a.where[id], 0);
    out[j] = id;
  }
}

// A page that a sequence has a copy of now is one sequence's less
__device__ __forceinline__ void copied(const Extension& a, int i) { atomicAdd(a.refs_out + a.moves.src[i], -1); }
__device__ __forceinline__ void copied(const Compaction&, int) {}

// Tables by blocks, `units` chunks of them, then what moves by warps
template <class P>
__global__ void __launch_bounds__(ROW_THREADS, 3)
finish_kernel(const P a, const Pools pools, int64_t units, int chunks) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) table_chunk(a, (int)(u / chunks), (int)(u % chunks) * CHUNK + threadIdx.x);
  const int n = *a.moves.n;
  for (int i = blockIdx.x * ROW_THREADS + threadIdx.x; i < n; i += gridDim.x * ROW_THREADS) copied(a, i);
  move<MANY_LOADS>(pools, a.page_size, a.moves.src, a.moves.dst, a.moves.rows, n, (int64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5), (int64_t)gridDim.x * (ROW_THREADS / 32));
}

// ---- host ----------------------------------------------------------------------------------------------------------
static int check_books(const void* table, int64_t ld, const void* lens, const void* refs, const void* table_out, int64_t ld_out, const void* refs_out, int B, int W,
                       int pages, int page_size) {
  if (B < 0 || W < 0 || W >= (1 << 29) || pages < 0 || pages > (1 << 28) || page_size <= 0 || page_size > (1 << 29)) return Q40_E_SHAPE;
  if (B > 0 && (!lens || (W > 0 && (!table || !table_out)))) return Q40_E_NULL;
  if (pages > 0 && (!refs || !refs_out)) return Q40_E_NULL;
  if (B > 1 && (ld < W || ld_out < W)) return Q40_E_SHAPE;
  if (!q40_aligned(table, 4) || !q40_aligned(lens, 4) || !q40_aligned(refs, 4) || !q40_aligned(table_out, 4) || !q40_aligned(refs_out, 4)) return Q40_E_ALIGN;
  return Q40_OK;
}
static void fill(Books& b, const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, int32_t* table_out, int64_t ld_out, int32_t* lens_out,
                 int32_t* refs_out, int B, int W, int pages, int page_size) {
  b.table = table; b.ld = ld; b.lens = lens; b.refs = refs;
  b.table_out = table_out; b.ld_out = ld_out; b.lens_out = lens_out; b.refs_out = refs_out;
  b.B = B; b.W = W; b.pages = pages; b.page_size = page_size; b.page_shift = page_shift_of(page_size);
}
static int fill_pools(Pools& p, void* k, void* v, float* ks, float* vs, int cache_type, int heads, int64_t P, int pages, int page_size) {
  if (cache_type < CACHE_F16 || cache_type > CACHE_E4M3) return Q40_E_UNSUPPORTED;
  if (heads < 0 || P < 0 || P > 0x7fffffffLL || (int64_t)pages * page_size > P || (cache_type != CACHE_F16 && P % page_size != 0)) return Q40_E_SHAPE;
  if (heads > 0 && pages > 0 && (!k || !v || (cache_type != CACHE_F16 && (!ks || !vs)))) return Q40_E_NULL;
  if (!q40_aligned(k, 16) || !q40_aligned(v, 16) || !q40_aligned(ks, 4) || !q40_aligned(vs, 4)) return Q40_E_ALIGN;
  p.k = (unsigned char*)k; p.v = (unsigned char*)v;
  p.ks = cache_type == CACHE_F16 ? nullptr : ks; p.vs = cache_type == CACHE_F16 ? nullptr : vs;
  p.heads = heads; p.row_bytes = ATTN_D * (cache_type == CACHE_F16 ? 2 : 1); p.P = P; p.scale_stride = P / page_size;
  return Q40_OK;
}
// A second launch of as many blocks as there is work for, at most `most_moves` pages to move
template <class P>
static cudaError_t finish(const P& a, const Pools& pools, int64_t most_moves, cudaStream_t st) {
  const int chunks = std::max(1, (a.W + CHUNK - 1) / CHUNK);
  const int64_t units = (int64_t)a.B * chunks, pieces = ((int64_t)a.page_size * pools.row_bytes + MANY_LOADS * 512 - 1) / (MANY_LOADS * 512);
  const int64_t warps = std::min<int64_t>(most_moves, 1 << 20) * std::min<int64_t>(2 * (int64_t)pools.heads * pieces, 1 << 20);
  const int64_t blocks = std::min<int64_t>(std::max<int64_t>(std::max(units, (warps + 7) / 8), 1), 148 * 3);
  return q40_launch_pdl(finish_kernel<P>, dim3((unsigned)blocks), dim3(ROW_THREADS), 0, st, a, pools, units, chunks);
}

// CTAs of 1024 threads for a plan that each makes for itself, with `rows` of W entries to write and up to most_moves pages to move: a warp for each piece, an SM for each CTA
static int few_ctas(const Books& b, const Pools& pools, int64_t most_moves) {
  const int64_t units = (int64_t)b.B * ((b.W + UNIT - 1) / UNIT), pieces = ((int64_t)b.page_size * pools.row_bytes + FEW_LOADS * 512 - 1) / (FEW_LOADS * 512);
  const int64_t warps = std::min<int64_t>(most_moves, 1 << 20) * std::min<int64_t>(2 * (int64_t)pools.heads * pieces, 1 << 20) + units;
  return (int)std::min<int64_t>(std::max<int64_t>((warps + WARPS - 1) / WARPS, 1), 148);
}
// In place that is one cluster, which should not have more to do than some hundred SMs would do in a second launch: up to
constexpr int MOST_IN_PLACE = 4 * CLUSTER;       // CTAs' worth of it
template <bool IN_PLACE, class P>
static cudaError_t launch_few(void (*kern)(P, Pools), const P& a, const Pools& pools, int ctas, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(IN_PLACE ? CLUSTER : ctas));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CLUSTER;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = IN_PLACE ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a, pools);
}
constexpr int EXTEND_FEW_SMEM = (8 * FEW_ROWS + 2 * FEW_PAGES) * (int)sizeof(int), COMPACT_FEW_SMEM = (2 * FEW_PAGES / 32 + FEW_PAGES + 2) * (int)sizeof(int);

// Forks whose entries the warps of one cluster hold
static bool fork_is_few(int B, int W, int n_pages) { return (int64_t)B * std::max(1, (W + UNIT - 1) / UNIT) <= CLUSTER * WARPS * FORK_UNITS && n_pages <= 1 << 16; }

static size_t extend_bytes(int B, int pages) { return ((size_t)B * 7 + 2 * (size_t)pages + 4) * sizeof(int); }
static size_t compact_bytes(int pages) { return (3 * ((size_t)pages / 2 + 1) + 4) * sizeof(int); }

}  // namespace books
}  // namespace q40

extern "C" size_t q40_page_fork_workspace_bytes(int B, int W, int n_pages) {
  using namespace q40::books;
  return B <= 0 || W < 0 || fork_is_few(B, W, n_pages) ? 0 : ((size_t)B * W + B) * sizeof(int);
}

extern "C" int q40_page_fork(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, const int32_t* parents, int32_t* table_out, int64_t ld_out,
                             int32_t* lens_out, int32_t* refs_out, int B, int W, int n_pages, int page_size, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::books;
  const int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (B > 0 && (!parents || !lens_out)) return Q40_E_NULL;
  if (!q40_aligned(parents, 4) || !q40_aligned(lens_out, 4) || !q40_aligned(workspace, 4)) return Q40_E_ALIGN;
  if (table == table_out && ld != ld_out && B > 1) return Q40_E_SHAPE;
  const int chunks = std::max(1, (W + CHUNK - 1) / CHUNK);
  if ((int64_t)B * chunks > 0x7fffffffLL) return Q40_E_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  Books b{};
  fill(b, table, ld, lens, refs, table_out, ld_out, lens_out, refs_out, B, W, n_pages, page_size);
  cudaError_t e = cudaSuccess;
  if (fork_is_few(B, W, n_pages)) {
    const int row_units = std::max(1, (W + UNIT - 1) / UNIT);
    if (B > 0 || (n_pages > 0 && refs != refs_out)) e = q40_launch_pdl(fork_few_kernel, dim3(CLUSTER), dim3(NT), 0, st, b, parents, B * row_units, row_units);
    return e == cudaSuccess ? Q40_OK : (int)e;
  }
  if (B > 0 && ((W > 0 && table == table_out) || lens == lens_out)) {          // sequences read each other's rows: as they were
    if (!workspace || workspace_bytes < q40_page_fork_workspace_bytes(B, W, n_pages)) return Q40_E_WORKSPACE;
    int32_t* const old = (int32_t*)workspace;
    if (W > 0) e = cudaMemcpy2DAsync(old, (size_t)W * 4, table, (size_t)(B > 1 ? ld : W) * 4, (size_t)W * 4, B, cudaMemcpyDeviceToDevice, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(old + (size_t)B * W, lens, (size_t)B * 4, cudaMemcpyDeviceToDevice, st);
    b.table = old;
    b.ld = W;
    b.lens = old + (size_t)B * W;
  }
  if (e == cudaSuccess && n_pages > 0 && refs != refs_out)
    e = q40_launch_pdl(fork_refs_kernel, dim3(std::min(592, (n_pages + 255) / 256)), dim3(256), 0, st, refs, refs_out, n_pages);
  if (e == cudaSuccess && B > 0) e = q40_launch_pdl(fork_rows_kernel, dim3((unsigned)(B * chunks)), dim3(ROW_THREADS), 0, st, b, parents, chunks);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

extern "C" size_t q40_page_extend_workspace_bytes(int B, int n_pages, int in_place) {
  using namespace q40::books;
  return B < 0 || n_pages < 0 || (!in_place && B <= FEW_ROWS && n_pages <= FEW_PAGES) ? 0 : extend_bytes(B, n_pages);
}

extern "C" int q40_page_extend(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, const int32_t* add, int32_t* table_out, int64_t ld_out,
                               int32_t* lens_out, int32_t* refs_out, int B, int W, int n_pages, int page_size, void* kpool, void* vpool, float* k_scale,
                               float* v_scale, int cache_type, int64_t P, int heads, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::books;
  int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (B > MOST_SEQUENCES) return Q40_E_SHAPE;
  if (B > 0 && (!add || !lens_out)) return Q40_E_NULL;
  if (!q40_aligned(add, 4) || !q40_aligned(lens_out, 4) || !q40_aligned(workspace, 16)) return Q40_E_ALIGN;
  Pools pools{};
  rc = fill_pools(pools, kpool, vpool, k_scale, v_scale, cache_type, heads, P, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (table == table_out && ld != ld_out && B > 1) return Q40_E_SHAPE;
  const bool some[3] = {B > 0 && W > 0, B > 0, n_pages > 0}, same[3] = {some[0] && table == table_out, some[1] && lens == lens_out, some[2] && refs == refs_out};
  const bool in_place = same[0] || same[1] || same[2], whole = same[0] == some[0] && same[1] == some[1] && same[2] == some[2];
  const bool few = B <= FEW_ROWS && n_pages <= FEW_PAGES && (!in_place || whole);
  if ((in_place || !few) && (!workspace || workspace_bytes < extend_bytes(B, n_pages))) return Q40_E_WORKSPACE;
  if (B == 0 && (n_pages == 0 || same[2])) return Q40_OK;
  Extension a{};
  fill(a, table, ld, lens, refs, table_out, ld_out, lens_out, refs_out, B, W, n_pages, page_size);
  a.add = add;
  const cudaStream_t st = (cudaStream_t)stream;
  const int ctas = few_ctas(a, pools, B);
  if (few && (!in_place || ctas <= MOST_IN_PLACE)) {
    static std::atomic<uint64_t> ready[2];
    const auto kern = in_place ? extend_few_kernel<true> : extend_few_kernel<false>;
    cudaError_t e = q40_allow_smem(ready[in_place], (const void*)kern, EXTEND_FEW_SMEM);
    const size_t smem = (8 * FEW_ROWS + 2 * (size_t)((n_pages + 3) / 4 * 4)) * sizeof(int);
    if (e == cudaSuccess) e = in_place ? launch_few<true, Additions>(kern, a, pools, ctas, smem, st) : launch_few<false, Additions>(kern, a, pools, ctas, smem, st);
    return e == cudaSuccess ? Q40_OK : (int)e;
  }
  a.plan = (int4*)workspace;
  int* const at = (int*)workspace + 4 * (size_t)B;
  a.moves = {at, at + 4, at + 4 + B, at + 4 + 2 * (size_t)B};
  a.writers = a.moves.rows + B;
  a.last = a.writers + n_pages;
  static std::atomic<uint64_t> ready;
  cudaError_t e = q40_allow_smem(ready, (const void*)extend_plan_kernel, (2 * MOST_SEQUENCES + 1) * (int)sizeof(int));
  if (e == cudaSuccess) e = q40_launch_pdl(extend_plan_kernel, dim3(CLUSTER), dim3(NT), (2 * (size_t)B + 1) * sizeof(int), st, a);
  if (e == cudaSuccess) e = finish(a, pools, B, st);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

extern "C" size_t q40_page_compact_workspace_bytes(int n_pages, int in_place) {
  using namespace q40::books;
  return n_pages < 0 || (!in_place && n_pages <= FEW_PAGES) ? 0 : compact_bytes(n_pages);
}

extern "C" int q40_page_compact(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, int32_t* table_out, int64_t ld_out, int32_t* refs_out,
                                int32_t* where, int B, int W, int n_pages, int page_size, void* kpool, void* vpool, float* k_scale, float* v_scale, int cache_type,
                                int64_t P, int heads, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::books;
  int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (n_pages > 0 && !where) return Q40_E_NULL;
  if (!q40_aligned(where, 4) || !q40_aligned(workspace, 16)) return Q40_E_ALIGN;
  Pools pools{};
  rc = fill_pools(pools, kpool, vpool, k_scale, v_scale, cache_type, heads, P, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (table == table_out && ld != ld_out && B > 1) return Q40_E_SHAPE;
  const bool in_place = (table == table_out && B > 0 && W > 0) || (refs == refs_out && n_pages > 0), few = n_pages <= FEW_PAGES;
  if ((in_place || !few) && (!workspace || workspace_bytes < compact_bytes(n_pages))) return Q40_E_WORKSPACE;
  Compaction a{};
  fill(a, table, ld, lens, refs, table_out, ld_out, nullptr, refs_out, B, W, n_pages, page_size);
  a.where = where;
  const size_t half = (size_t)n_pages / 2 + 1;
  const cudaStream_t st = (cudaStream_t)stream;
  const int ctas = few_ctas(a, pools, n_pages / 2);
  if (few && (!in_place || ctas <= MOST_IN_PLACE)) {
    static std::atomic<uint64_t> ready[2];
    const auto kern = in_place ? compact_few_kernel<true> : compact_few_kernel<false>;
    cudaError_t e = q40_allow_smem(ready[in_place], (const void*)kern, COMPACT_FEW_SMEM);
    const size_t smem = (2 * FEW_PAGES / 32 + 2 * half) * sizeof(int);
    if (e == cudaSuccess) e = in_place ? launch_few<true, Moving>(kern, a, pools, ctas, smem, st) : launch_few<false, Moving>(kern, a, pools, ctas, smem, st);
    return e == cudaSuccess ? Q40_OK : (int)e;
  }
  int* const at = (int*)workspace;
  a.moves = {at, at + 4, at + 4 + half, nullptr};
  a.old_refs = at + 4 + 2 * half;
  cudaError_t e = q40_launch_pdl(compact_plan_kernel, dim3(CLUSTER), dim3(NT), 0, st, a);
  if (e == cudaSuccess) e = finish(a, pools, n_pages / 2, st);
  return e == cudaSuccess ? Q40_OK : (int)e;
}
