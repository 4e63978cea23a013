// The pages of a paged cache: which sequences list them, and where they lie.  Sequences fork (q40_page_fork), get pages for their next tokens or give some back
// (q40_page_extend), and pages in use move to the front of their pools (q40_page_compact), by what the device's books say: a table of page ids and a length for
// each sequence, and for each page how many sequences list it (0: it is free).  Nothing goes by way of the host, so that a captured step can be replayed.
//
// Free pages are handed out in ascending order, to the sequences in theirs: results do not depend on which thread comes first.  A plan is made by one cluster of eight
// CTAs: each warp has a run of pages, which it counts through by ballots, the CTAs hand each other their sums through distributed shared memory, and a page that is the
// r-th free one looks up the sequence that wants it in the sums of what they want.  A second launch, of all SMs, writes the tables and moves what the pools hold.
//
// What bounds it: few sequences, the plan's chain of loads and three cluster barriers; pools that move, HBM.
#include <cooperative_groups.h>

#include <algorithm>

#include "pages_common.cuh"

namespace q40 {
namespace books {

namespace cg = cooperative_groups;

constexpr int CLUSTER = 8, NT = 1024, WARPS = NT / 32;      // of a plan
constexpr int MOST_SEQUENCES = 16384;                       // of an extension: what they want is summed in shared memory
constexpr int CHUNK = 1024, ROW_THREADS = 256;              // entries of a table that a block takes at a time
constexpr int PIECE = 4096;                                 // bytes that a warp copies at a time

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

// ---- forks ---------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
fork_refs_kernel(const int32_t* refs, int32_t* out, int n) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) out[i] = refs[i];
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
    const int id = j < n_new ? from[j] : 0;
    out[j] = id;
    if (p == row) continue;
    const int old = j < n_old ? own[j] : -1, now = j < n_new ? id : -1;
    if (old == now) continue;                            // a page that both list
    if (b.valid(now)) atomicAdd(b.refs_out + now, 1);
    if (b.valid(old)) atomicAdd(b.refs_out + old, -1);
  }
}

// ---- what plans share ----------------------------------------------------------------------------------------------
// A warp's run of pages, in order over the cluster
struct Run {
  int lo, hi;
  __device__ __forceinline__ Run(int pages, int rank) {
    const int each = ((pages + CLUSTER * WARPS - 1) / (CLUSTER * WARPS) + 31) / 32 * 32;
    const int64_t first = (int64_t)(rank * WARPS + (int)(threadIdx.x >> 5)) * each;
    lo = (int)min(first, (int64_t)pages);
    hi = (int)min(first + each, (int64_t)pages);
  }
};
// The pages of a run, 32 at a time, four of these requested together: f(first page, this lane's references; 0 behind the end)
template <class F>
__device__ __forceinline__ void through(const int32_t* refs, const Run& run, F f) {
  const int lane = threadIdx.x & 31;
  for (int p0 = run.lo; p0 < run.hi; p0 += 128) {
    int r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = p0 + 32 * i + lane < run.hi ? refs[p0 + 32 * i + lane] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + 32 * i < run.hi) f(p0 + 32 * i, r[i]);
  }
}
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
struct Extension : Books {
  const int32_t* add;
  int *writers, *last;               // of each page: sequences that write to it behind its rows, and the last of them
  int4* plan;                        // of each sequence: entries that stay, entries in all, entries before, length
  Moves moves;
};

struct Growth {
  int n, m, n0, n1;                  // tokens and pages, before and after
  int tail, shared;                  // a page that is in part filled and will be written to (-1: none), and its references
  bool grows;                        // into pages that the table has room for
  __device__ __forceinline__ Growth(const Extension& a, int b) {
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
  int* const info = wanted + a.B + 1;            // [B] PAGES: how many before; GROWS, WANTS any page, COPIES one
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
  const Run run(a.pages, rank);
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
      bool copies = false;
      if (g.grows) {
        // of sequences that all write to a page which no other lists, the last keeps it
        copies = g.tail >= 0 && g.shared > 1 && !(__ldcg(a.writers + g.tail) == g.shared && __ldcg(a.last + g.tail) == b);
        need = g.n1 - g.n0 + (copies ? 1 : 0);
      }
      info[b] = g.n0 | (g.grows ? GROWS : 0) | (need ? WANTS : 0) | (copies ? COPIES : 0);
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

// ---- compaction ----------------------------------------------------------------------------------------------------
struct Compaction : Books {
  int32_t* where;                    // [pages] a page's new id, or -1 (free)
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
  const Run run(a.pages, rank);
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

// Tables by blocks, `units` chunks of them, then what moves by warps: of each page and head, keys or values, PIECE bytes at a time
template <class P>
__global__ void __launch_bounds__(ROW_THREADS)
finish_kernel(const P a, const Pools pools, int64_t units, int chunks) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) table_chunk(a, (int)(u / chunks), (int)(u % chunks) * CHUNK + threadIdx.x);
  const int n = *a.moves.n, lane = threadIdx.x & 31;
  for (int i = blockIdx.x * ROW_THREADS + threadIdx.x; i < n; i += gridDim.x * ROW_THREADS) copied(a, i);
  const int pieces = (int)(((int64_t)a.page_size * pools.row_bytes + PIECE - 1) / PIECE);
  const int64_t per = (int64_t)2 * pools.heads * pieces, step = (int64_t)gridDim.x * (ROW_THREADS / 32);
  const int64_t at = (int64_t)blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5);
  int64_t i = at / per, rest = at % per;
  const int64_t i_step = step / per, rest_step = step % per;
  while (i < n) {
    const int src = a.moves.src[i], dst = a.moves.dst[i], piece = (int)(rest % pieces);
    const int64_t bytes = (int64_t)(a.moves.rows ? a.moves.rows[i] : a.page_size) * pools.row_bytes;
    int head = (int)(rest / pieces);
    const bool values = head >= pools.heads;
    if (values) head -= pools.heads;
    unsigned char* const pool = (values ? pools.v : pools.k) + (int64_t)head * pools.P * pools.row_bytes;
    const unsigned char* const from = pool + (int64_t)src * a.page_size * pools.row_bytes;
    unsigned char* const to = pool + (int64_t)dst * a.page_size * pools.row_bytes;
    uint4 x[PIECE / 512];
#pragma unroll
    for (int c = 0; c < PIECE / 512; ++c) {
      const int64_t off = (int64_t)piece * PIECE + c * 512 + lane * 16;
      if (off < bytes) x[c] = *reinterpret_cast<const uint4*>(from + off);
    }
    if (piece == 0 && lane == 0 && pools.ks) {
      float* const scale = (values ? pools.vs : pools.ks) + (int64_t)head * pools.scale_stride;
      scale[dst] = scale[src];
    }
#pragma unroll
    for (int c = 0; c < PIECE / 512; ++c) {
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
  const int64_t units = (int64_t)a.B * chunks, pieces = ((int64_t)a.page_size * pools.row_bytes + PIECE - 1) / PIECE;
  const int64_t warps = std::min<int64_t>(most_moves, 1 << 20) * std::min<int64_t>(2 * (int64_t)pools.heads * pieces, 1 << 20);
  const int64_t blocks = std::min<int64_t>(std::max<int64_t>(std::max(units, (warps + 7) / 8), 1), 148 * 3);
  return q40_launch_pdl(finish_kernel<P>, dim3((unsigned)blocks), dim3(ROW_THREADS), 0, st, a, pools, units, chunks);
}

static size_t extend_bytes(int B, int pages) { return ((size_t)B * 7 + 2 * (size_t)pages + 4) * sizeof(int); }
static size_t compact_bytes(int pages) { return (3 * ((size_t)pages / 2 + 1) + 4) * sizeof(int); }

}  // namespace books
}  // namespace q40

extern "C" int q40_page_fork(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, const int32_t* parents, int32_t* table_out, int64_t ld_out,
                             int32_t* lens_out, int32_t* refs_out, int B, int W, int n_pages, int page_size, void* stream) {
  using namespace q40::books;
  const int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (B > 0 && (!parents || !lens_out)) return Q40_E_NULL;
  if (!q40_aligned(parents, 4) || !q40_aligned(lens_out, 4)) return Q40_E_ALIGN;
  if (B > 0 && ((W > 0 && table == table_out) || lens == lens_out)) return Q40_E_UNSUPPORTED;
  Books b{};
  fill(b, table, ld, lens, refs, table_out, ld_out, lens_out, refs_out, B, W, n_pages, page_size);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (n_pages > 0 && refs != refs_out)
    e = q40_launch_pdl(fork_refs_kernel, dim3(std::min(592, (n_pages + 255) / 256)), dim3(256), 0, st, refs, refs_out, n_pages);
  const int chunks = std::max(1, (W + CHUNK - 1) / CHUNK);
  if ((int64_t)B * chunks > 0x7fffffffLL) return Q40_E_SHAPE;
  if (e == cudaSuccess && B > 0) e = q40_launch_pdl(fork_rows_kernel, dim3((unsigned)(B * chunks)), dim3(ROW_THREADS), 0, st, b, parents, chunks);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

extern "C" size_t q40_page_extend_workspace_bytes(int B, int n_pages) { return B < 0 || n_pages < 0 ? 0 : q40::books::extend_bytes(B, n_pages); }

extern "C" int q40_page_extend(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, const int32_t* add, int32_t* table_out, int64_t ld_out,
                               int32_t* lens_out, int32_t* refs_out, int B, int W, int n_pages, int page_size, void* kpool, void* vpool, float* k_scale,
                               float* v_scale, int cache_type, int64_t P, int heads, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::books;
  int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (B > MOST_SEQUENCES) return Q40_E_SHAPE;
  if (!workspace || (B > 0 && (!add || !lens_out))) return Q40_E_NULL;
  if (!q40_aligned(add, 4) || !q40_aligned(lens_out, 4) || !q40_aligned(workspace, 16)) return Q40_E_ALIGN;
  Pools pools{};
  rc = fill_pools(pools, kpool, vpool, k_scale, v_scale, cache_type, heads, P, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (workspace_bytes < extend_bytes(B, n_pages)) return Q40_E_WORKSPACE;
  if (table == table_out && ld != ld_out && B > 1) return Q40_E_SHAPE;
  if (B == 0 && (n_pages == 0 || refs == refs_out)) return Q40_OK;
  Extension a{};
  fill(a, table, ld, lens, refs, table_out, ld_out, lens_out, refs_out, B, W, n_pages, page_size);
  a.add = add;
  a.plan = (int4*)workspace;
  int* at = (int*)workspace + 4 * (size_t)B;
  a.moves = {at, at + 4, at + 4 + B, at + 4 + 2 * (size_t)B};
  a.writers = a.moves.rows + B;
  a.last = a.writers + n_pages;
  static std::atomic<uint64_t> ready;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = q40_allow_smem(ready, (const void*)extend_plan_kernel, (2 * MOST_SEQUENCES + 1) * (int)sizeof(int));
  if (e == cudaSuccess) e = q40_launch_pdl(extend_plan_kernel, dim3(CLUSTER), dim3(NT), (2 * (size_t)B + 1) * sizeof(int), st, a);
  if (e == cudaSuccess) e = finish(a, pools, B, st);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

extern "C" size_t q40_page_compact_workspace_bytes(int n_pages) { return n_pages < 0 ? 0 : q40::books::compact_bytes(n_pages); }

extern "C" int q40_page_compact(const int32_t* table, int64_t ld, const int32_t* lens, const int32_t* refs, int32_t* table_out, int64_t ld_out, int32_t* refs_out,
                                int32_t* where, int B, int W, int n_pages, int page_size, void* kpool, void* vpool, float* k_scale, float* v_scale, int cache_type,
                                int64_t P, int heads, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::books;
  int rc = check_books(table, ld, lens, refs, table_out, ld_out, refs_out, B, W, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (!workspace || (n_pages > 0 && !where)) return Q40_E_NULL;
  if (!q40_aligned(where, 4) || !q40_aligned(workspace, 16)) return Q40_E_ALIGN;
  Pools pools{};
  rc = fill_pools(pools, kpool, vpool, k_scale, v_scale, cache_type, heads, P, n_pages, page_size);
  if (rc != Q40_OK) return rc;
  if (workspace_bytes < compact_bytes(n_pages)) return Q40_E_WORKSPACE;
  if (table == table_out && ld != ld_out && B > 1) return Q40_E_SHAPE;
  Compaction a{};
  fill(a, table, ld, lens, refs, table_out, ld_out, nullptr, refs_out, B, W, n_pages, page_size);
  a.where = where;
  int* const at = (int*)workspace;
  const size_t half = (size_t)n_pages / 2 + 1;
  a.moves = {at, at + 4, at + 4 + half, nullptr};
  a.old_refs = at + 4 + 2 * half;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = q40_launch_pdl(compact_plan_kernel, dim3(CLUSTER), dim3(NT), 0, st, a);
  if (e == cudaSuccess) e = finish(a, pools, n_pages / 2, st);
  return e == cudaSuccess ? Q40_OK : (int)e;
}
