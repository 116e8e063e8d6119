// Block tables, slots and offsets of a step from its requests' lengths, on the GPU, with the pages they take from a stack of
// free ones; and pages given back.
//
// plan: request i adds new[i] tokens to sequence rows[i]. It needs need_i = ceil((past + new) / page) - ceil(past / page) pages and
// is taken if it needs none, or if the requests up to it need no more than are free; the k-th page of a request that is taken
// is so far below the stack's top as pages were given out before it. Everything else follows from prefix sums over the requests:
// a token finds its request by bisection of the offsets, its page in the sequence's table row or, past what that held before, in
// the stack itself.
//
// A few kilobytes go through it, so a call is latency: one launch, every CTA forming the same prefix sums in shared memory (16
// bytes a request) and then writing its share of tokens and table entries. Nothing that the sums read is written before the last
// CTA has read it: that CTA, found by a counter, writes the new lengths and the stack's size. (New table entries lie behind those
// that are read, pages given back above the stack's top.) Plan and trim of 64 requests of a token take 12.3 us in a graph, of 256 requests of 0 to
// 512 tokens 17.1.

#include "common.cuh"
#include "attention.cuh"
#include "paged_plan.cuh"

namespace omni {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// The exclusive sum over the threads before this one of v, and over all of them.
OMNI_DEV int64_t block_scan(int64_t v, int64_t* total, int64_t* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (part may still be read)
  if (lane == 31) part[warp] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int64_t p = part[w];
    if (w < warp) before += p;
    all += p;
  }
  *total = all;
  return before + x - v;
}

OMNI_DEV uint32_t hash(uint32_t x) { return x * 0x9e3779b9u; }

struct Request {
  int row;    // the sequence, -1: refused
  int past;   // its positions before the step (0 where it has no sequence)
  int first;  // its first token (plan); pages given back after its own (trim)
  int start;  // pages given out before its own (plan)
};

// Dynamic shared memory: requests, then the table of sequences (a power of two of at least twice the requests).
OMNI_DEV int slots_of(int requests) {
  int n = 32;
  while (n < 2 * requests) n *= 2;
  return n;
}
size_t smem_bytes(int requests) {
  int n = 32;
  while (n < 2 * requests) n *= 2;
  return (size_t)requests * sizeof(Request) + (size_t)n * sizeof(int);
}

// Enters request i into the table of sequences: of several of one sequence the first stays. Its place, or -1.
OMNI_DEV int enter(int* seen, int n, const Request* req, int row, int i) {
  int at = (int)(hash((uint32_t)row) >> 8) & (n - 1);
  for (int k = 0; k < n; ++k) {
    const int old = atomicCAS(seen + at, -1, i);
    if (old == -1) return at;
    if (req[old].row == row) {
      atomicMin(seen + at, i);
      return at;
    }
    at = (at + 1) & (n - 1);
  }
  return -1;
}

// The last request of [0, n) with key(r) <= x; key ascends and key(0) <= x.
template <typename F>
OMNI_DEV int last_at_most(int n, F key, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (key(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Common to both: rows and their first requests. Returns through req the sequence or -1, and past; per thread the items
// [i0, i1).
OMNI_DEV void read_requests(const PlanArgs& a, Request* req, int* seen, int n, int i0, int i1) {
  for (int i = threadIdx.x; i < n; i += kThreads) seen[i] = -1;
  for (int i = i0; i < i1; ++i) {
    const int64_t r = a.rows[i];
    req[i].row = r >= 0 && r < a.s.seqs ? (int)r : -1;
  }
  __syncthreads();
  for (int i = i0; i < i1; ++i) req[i].start = req[i].row >= 0 ? enter(seen, n, req, req[i].row, i) : -1;
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    const int at = req[i].start;
    const int64_t past = req[i].row >= 0 ? a.s.length[req[i].row] : 0;
    const bool ok = past >= 0 && past <= (int64_t)a.s.table_width * a.s.page;
    req[i].past = ok ? (int)past : 0;
    if (at < 0 || seen[at] != i || !ok) {
      raise_status(a.status, kStatusIndex);
      req[i].start = -1;  // refused
    }
  }
}

// Whether this CTA is the last that has read the state.
OMNI_DEV bool last_reader(unsigned* arrivals) {
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(arrivals, 1u) == gridDim.x - 1;
    if (last) {
      *arrivals = 0u;
      __threadfence();
    }
  }
  __syncthreads();
  return last;
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int64_t part[kWarps];
  Request* req = reinterpret_cast<Request*>(smem);
  int* seen = reinterpret_cast<int*>(smem + (size_t)a.requests * sizeof(Request));
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = a.requests, page = a.s.page;
  const int per = (b + kThreads - 1) / kThreads;
  const int i0 = min(b, (int)threadIdx.x * per), i1 = min(b, i0 + per);
  int64_t count = *a.s.count;
  if (count < 0 || count > a.s.pages) {
    if (threadIdx.x == 0) raise_status(a.status, kStatusIndex);
    count = 0;
  }
  read_requests(a, req, seen, slots_of(b), i0, i1);
  const int64_t room = (int64_t)min(a.s.table_width, a.batch_width) * page;  // positions that the tables have entries for

  // A request's tokens, whether it stays, and the pages it needs.
  auto fresh = [&](int i) { return max((int64_t)0, a.want[i]); };
  auto pages = [&](int n) { return (n + page - 1) / page; };
  int64_t q = 0, need = 0, q_all, need_all, k_all;
  for (int i = i0; i < i1; ++i) q += min(fresh(i), (int64_t)0x7fffffff);
  int64_t q_at = block_scan(q, &q_all, part);
  for (int i = i0; i < i1; ++i) {
    const int64_t n = fresh(i), end = q_at + min(n, (int64_t)0x7fffffff);
    bool ok = req[i].start >= 0;
    if (a.want[i] < 0 || end > a.tokens) {
      ok = false;
      raise_status(a.status, kStatusIndex);
    }
    if (ok && req[i].past + n > room) ok = false;
    req[i].first = (int)min(q_at, (int64_t)a.tokens);
    q_at = end;
    if (!ok) req[i].start = -1;
    else {
      req[i].start = pages(req[i].past + (int)n) - pages(req[i].past);
      need += req[i].start;
    }
  }
  int64_t need_at = block_scan(need, &need_all, part);
  int64_t k = 0;
  for (int i = i0; i < i1; ++i) {
    const int mine = req[i].start;
    bool ok = mine >= 0;
    if (mine > 0) {
      need_at += mine;
      ok = need_at <= count;
    }
    if (!ok) req[i].row = -1 - (req[i].row + 1);  // refused: the sequence stays readable as -2 - row (none: -1)
    req[i].start = ok ? (int)(need_at - mine) : 0;
    k += req[i].past + (ok ? fresh(i) : 0);
  }
  int64_t k_at = block_scan(k, &k_all, part);
  if (blockIdx.x == 0) {
    for (int i = i0; i < i1; ++i) {
      const bool ok = req[i].row >= 0;
      a.q_offsets[i] = req[i].first;
      a.k_offsets[i] = k_at;
      a.lengths[i] = ok ? req[i].past + 1 : 0;
      a.taken[i] = ok;
      k_at += req[i].past + (ok ? fresh(i) : 0);
    }
    if (threadIdx.x == 0) {
      a.q_offsets[b] = min(q_all, (int64_t)a.tokens);
      a.k_offsets[b] = k_all;
    }
  }
  __syncthreads();

  // The tokens.
  const int at = blockIdx.x * kThreads + threadIdx.x, step = gridDim.x * kThreads;
  auto stack = [&](const Request& r, int j) { return a.s.free[count - 1 - (r.start + j)]; };
  const int q_end = (int)min(q_all, (int64_t)a.tokens);
  for (int t = at; t < a.tokens; t += step) {
    int64_t pos = 0, slot = -1;
    if (t < q_end) {
      const Request r = req[last_at_most(b, [&](int i) { return (int64_t)req[i].first; }, t)];
      const int p = r.past + (t - r.first);
      pos = p;
      if (r.row >= 0) {
        const int pi = p / page, held = pages(r.past);
        const int64_t id = pi < held ? a.s.table[r.row * a.s.table_stride + pi] : stack(r, pi - held);
        slot = id * page + (p - pi * page);
      } else {
        pos = min(p, a.last);
      }
    }
    a.pos[t] = pos;
    a.slots[t] = slot;
  }
  // The batch's table, and the sequences' new entries.
  const int64_t entries = (int64_t)b * a.batch_width;
  for (int64_t e = at; e < entries; e += step) {
    const int i = (int)((uint32_t)e / (uint32_t)a.batch_width), j = (int)((uint32_t)e - (uint32_t)i * (uint32_t)a.batch_width);
    const Request r = req[i];
    const int row = r.row >= 0 ? r.row : -2 - r.row;  // (-1: no sequence)
    const int held = row >= 0 ? pages(r.past) : 0;
    int32_t id = 0;
    if (j < held) {
      id = a.s.table[row * a.s.table_stride + j];
    } else if (r.row >= 0 && j < pages(r.past + (int)fresh(i))) {
      id = stack(r, j - held);
      a.s.table[row * a.s.table_stride + j] = id;
    }
    a.batch_table[e] = id;
  }
  if (last_reader(a.arrivals)) {
    int64_t got = 0, all;
    for (int i = i0; i < i1; ++i)
      if (req[i].row >= 0) {
        const int n = (int)fresh(i);
        got += pages(req[i].past + n) - pages(req[i].past);
        a.s.length[req[i].row] = req[i].past + n;
      }
    block_scan(got, &all, part);
    if (threadIdx.x == 0) *a.s.count = count - all;
  }
}

// The pages past what is kept go back, the last request's first and each request's last page first: as plan took them, so that a
// trim to the lengths before a plan leaves the stack as that found it.
__global__ void __launch_bounds__(kThreads) trim_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int64_t part[kWarps];
  Request* req = reinterpret_cast<Request*>(smem);
  int* seen = reinterpret_cast<int*>(smem + (size_t)a.requests * sizeof(Request));
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = a.requests, page = a.s.page;
  const int per = (b + kThreads - 1) / kThreads;
  const int i0 = min(b, (int)threadIdx.x * per), i1 = min(b, i0 + per);
  int64_t count = *a.s.count;
  bool sound = count >= 0 && count <= a.s.pages;
  read_requests(a, req, seen, slots_of(b), i0, i1);
  auto pages = [&](int n) { return (n + page - 1) / page; };
  int64_t give = 0, all;
  for (int i = i0; i < i1; ++i) {
    const int64_t keep = a.want[i];
    if (req[i].start >= 0 && (keep < 0 || keep > req[i].past)) {
      raise_status(a.status, kStatusIndex);
      req[i].start = -1;
    }
    req[i].start = req[i].start >= 0 ? pages(req[i].past) - pages((int)keep) : -1;
    if (req[i].start > 0) give += req[i].start;
  }
  int64_t g_at = block_scan(give, &all, part);
  for (int i = i0; i < i1; ++i) {
    req[i].first = (int)min(g_at, (int64_t)0x7fffffff);
    if (req[i].start > 0) g_at += req[i].start;
  }
  if (sound && count + all > a.s.pages) sound = false;  // more pages than there are: nothing goes back
  if (!sound && threadIdx.x == 0) raise_status(a.status, kStatusIndex);
  __syncthreads();
  if (sound) {
    for (int64_t t = blockIdx.x * kThreads + threadIdx.x; t < all; t += gridDim.x * kThreads) {
      const Request r = req[last_at_most(b, [&](int i) { return (int64_t)req[i].first; }, t)];
      const int j = pages(r.past) - r.start + (int)(t - r.first);  // page j of its sequence: the t-th from the stack's new top
      a.s.free[count + all - 1 - t] = a.s.table[r.row * a.s.table_stride + j];
    }
  }
  if (last_reader(a.arrivals) && sound) {
    for (int i = i0; i < i1; ++i)
      if (req[i].start >= 0) a.s.length[req[i].row] = a.want[i];
    if (threadIdx.x == 0) *a.s.count = count + all;
  }
}

int ctas(int64_t work) {
  const int64_t n = (work + 2 * kThreads - 1) / (2 * kThreads), most = device_sm_count();
  return (int)(n < 1 ? 1 : n > most ? most : n);
}

}  // namespace

cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t stream) {
  static PerDevice done;
  const size_t bytes = smem_bytes(a.requests);
  if (cudaError_t e = allow_smem(plan_kernel, (int)smem_bytes(kPlanMaxRequests), done)) return e;
  const int64_t work = (int64_t)a.tokens + (int64_t)a.requests * a.batch_width;
  return launch_dependent(plan_kernel, dim3((unsigned)ctas(work)), dim3(kThreads), bytes, stream, a);
}

cudaError_t launch_paged_trim(const PlanArgs& a, cudaStream_t stream) {
  static PerDevice done;
  const size_t bytes = smem_bytes(a.requests);
  if (cudaError_t e = allow_smem(trim_kernel, (int)smem_bytes(kPlanMaxRequests), done)) return e;
  // (How many pages go back is known on the device alone: a CTA for every 64 requests.)
  return launch_dependent(trim_kernel, dim3((unsigned)ctas((int64_t)a.requests * 16)), dim3(kThreads), bytes, stream, a);
}

}  // namespace omni
