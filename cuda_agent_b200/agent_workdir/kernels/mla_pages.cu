// Pages of the latent cache: copied, taken for longer sequences, shared by forks, given back, moved together.
//
// A page is free when its reference count is 0, and free pages are always taken lowest number first. That rule
// needs no list to be kept beside the counts, makes every result independent of the order in which CTAs run,
// and keeps the used part of a pool dense.
//
// The decisions of a call (which pages, is there room, is the list sound) are made by one CTA that scans the
// counts, 4096 at a time, and stops when it has found enough. extend and fork change nothing before they are all made, or
// nothing at all; copy leaves out the pairs it refuses, free and compact the table entries that they find wrong on their way. The
// bulk (page data, table rows) is done by the whole device in a second launch, which reads what was decided from
// scratch memory, so the host never waits. Page data is bound by memory: 16 bytes per access, 64 per thread in
// flight.
// Measured: the compaction of a pool of 2048 pages of 64 rows x 8 layers, half of them in use, 95 us for the pages that move (582 MB,
// 6.1 TB/s) and 5.2 us to decide; 4 forks of a 1500-row sequence 5.5 us to decide and 2.8 us to carry out; 200 sequences
// of 8192 rows and less given back in 3.4 us.
#include "cab_common.cuh"

namespace {

constexpr int kPlan = 1024;                    // threads of the deciding CTA
constexpr int kCopy = 256;
constexpr int kScan = 4;                       // counts per thread and step of a scan

// Scratch, in ints: [16] what was decided, then three arrays of num_pages and three of n + 1.
struct Scratch {
  int* head;                                   // [0] pages to copy, [1] the call is carried out
  int *list_a, *list_b, *map;                  // num_pages each
  int *n_a, *n_b, *n_c;                        // n + 1 each
};
size_t scratch_ints(int num_pages, int n) { return 16 + 3 * (size_t)num_pages + 3 * ((size_t)n + 1); }
Scratch carve(void* scratch, int num_pages, int n) {
  int* p = static_cast<int*>(scratch);
  Scratch s;
  s.head = p;
  s.list_a = p + 16; s.list_b = s.list_a + num_pages; s.map = s.list_b + num_pages;
  s.n_a = s.map + num_pages; s.n_b = s.n_a + n + 1; s.n_c = s.n_b + n + 1;
  return s;
}

struct Pool {
  int *table, *length, *refcount;
  int slots, max_pages, num_pages, page_size;
};

__device__ __forceinline__ void raise(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}
__device__ __forceinline__ int pages_for(int rows, int page_size) { return (int)(((long long)rows + page_size - 1) / page_size); }

// Exclusive scan over the 1024 threads of the deciding CTA; `total` gets the sum.
template <typename N>
__device__ __forceinline__ N plan_scan(N v, N& total) {
  __shared__ N warps[kPlan / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  N x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  if (warp == 0) {
    N w = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const N y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warps[lane] = w;
  }
  __syncthreads();
  total = warps[kPlan / 32 - 1];
  return x - v + (warp ? warps[warp - 1] : 0);
}

// The `want` lowest free pages to list[0 .. want), ascending. Returns whether there are as many.
__device__ bool lowest_free(const int* refcount, int num_pages, int want, int* list) {
  int found = 0;
  for (int base = 0; base < num_pages && found < want; base += kPlan * kScan) {
    const int p0 = base + threadIdx.x * kScan;
    bool is[kScan];
    int mine = 0, total;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      is[k] = p0 + k < num_pages && refcount[p0 + k] == 0;
      mine += is[k];
    }
    int at = found + plan_scan(mine, total);
#pragma unroll
    for (int k = 0; k < kScan; ++k)
      if (is[k]) {
        if (at < want) list[at] = p0 + k;
        ++at;
      }
    found += total;
  }
  return found >= want;
}

// ------------------------------------------------------------------------------------------------ copy
// Sound pairs to n_a -> n_b, -1 for the others. The marks of the pages named are set up here, so `map` may hold
// anything on entry.
__global__ void __launch_bounds__(kPlan) mla_pages_check_copy_kernel(const int* src, const int* dst, int n, int num_pages,
                                                                     Scratch s, int* status) {
  cab::after_predecessor();
  constexpr int kSrc = 1, kDst = 2, kTwice = 4;
  if (threadIdx.x == 0 && status) *status = 0;
  if (threadIdx.x == 0) s.head[0] = n;
  auto real = [&](int a, int b) { return a >= 0 && b >= 0 && a < num_pages && b < num_pages && a != b; };
  for (int i = threadIdx.x; i < n; i += kPlan)
    if (real(src[i], dst[i])) s.map[src[i]] = s.map[dst[i]] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan)
    if (real(src[i], dst[i])) {
      atomicOr(s.map + src[i], kSrc);
      if (atomicOr(s.map + dst[i], kDst) & kDst) atomicOr(s.map + dst[i], kTwice);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int a = src[i], b = dst[i];
    bool ok = real(a, b);
    if (ok && ((s.map[b] & (kSrc | kTwice)) || (s.map[a] & kDst))) {
      ok = false;
      raise(status, CAB_PAGED_BAD_INDEX);
    } else if (a >= 0 && b >= 0 && (a >= num_pages || b >= num_pages)) {
      raise(status, CAB_PAGED_BAD_INDEX);
    }
    s.n_a[i] = ok ? a : -1;
    s.n_b[i] = ok ? b : -1;
  }
}

// pages[:, dst[i]] = pages[:, src[i]] for i < head[0]; `from` < 0 skips. A CTA's share is pieces of 4 * 256 units.
template <typename Unit>
__device__ __forceinline__ void copy_pages(uint8_t* pages, long long layer_stride, int layers, long long page_bytes, int count,
                                           const int* src, const int* dst) {
  const long long units = page_bytes / (long long)sizeof(Unit);
  const int pieces = (int)((units + 4 * kCopy - 1) / (4 * kCopy));
  const long long total = (long long)count * layers * pieces;
  for (long long e = blockIdx.x; e < total; e += gridDim.x) {
    const int piece = (int)(e % pieces);
    const long long rest = e / pieces;
    const int layer = (int)(rest % layers), i = (int)(rest / layers);
    const int a = src[i], b = dst[i];
    if (a < 0 || b < 0) continue;
    const Unit* from = reinterpret_cast<const Unit*>(pages + layer * layer_stride + a * page_bytes);
    Unit* to = reinterpret_cast<Unit*>(pages + layer * layer_stride + b * page_bytes);
    const long long u0 = (long long)piece * 4 * kCopy + threadIdx.x;
    Unit v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (u0 + k * kCopy < units) v[k] = from[u0 + k * kCopy];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (u0 + k * kCopy < units) to[u0 + k * kCopy] = v[k];
  }
}

template <typename Unit>
__global__ void __launch_bounds__(kCopy) mla_pages_copy_kernel(uint8_t* pages, long long layer_stride, int layers,
                                                               long long page_bytes, const int* count, const int* src,
                                                               const int* dst) {
  cab::after_predecessor();
  copy_pages<Unit>(pages, layer_stride, layers, page_bytes, *count, src, dst);
}

// ------------------------------------------------------------------------------------------------ extend
// n_a: the present length of sequence i, n_b: pages needed before i, n_c: whether i's length was
// exchanged for the mark that finds a sequence listed twice.
__global__ void __launch_bounds__(kPlan) mla_pages_extend_kernel(Pool q, const int* seqs, const int* new_length, int n,
                                                                 Scratch s, int* status) {
  cab::after_predecessor();
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const long long most = (long long)q.max_pages * q.page_size;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int seq = seqs[i];
    s.n_c[i] = 0;
    if ((unsigned)seq >= (unsigned)q.slots) { atomicMax(&bad, (int)CAB_PAGED_BAD_INDEX); continue; }
    const int old = atomicExch(q.length + seq, -1);
    if (old < 0) { atomicMax(&bad, (int)CAB_PAGED_BAD_INDEX); continue; }   // listed before (or never a length)
    s.n_a[i] = old;
    s.n_c[i] = 1;
    if (new_length[i] > most) atomicMax(&bad, (int)CAB_PAGED_NO_ROOM);
  }
  __syncthreads();
  int want = 0;
  bool room = true;
  if (!bad) {
    for (int base = 0; base < n; base += kPlan) {
      const int i = base + threadIdx.x;
      long long need = 0, total;
      if (i < n) need = max(0, pages_for(new_length[i], q.page_size) - pages_for(s.n_a[i], q.page_size));
      const long long at = want + plan_scan(need, total);
      if (i < n) s.n_b[i] = (int)min(at, q.num_pages + 1LL);
      want = (int)min(want + total, q.num_pages + 1LL);      // more than there are: refused below
    }
    room = want <= q.num_pages && lowest_free(q.refcount, q.num_pages, want, s.list_a);
    __syncthreads();
  }
  const bool go = !bad && room;
  if (go) {
    for (int k = threadIdx.x; k < want; k += kPlan) {
      int lo = 0, hi = n;                      // last i with n_b[i] <= k
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.n_b[mid] <= k) lo = mid; else hi = mid;
      }
      const int page = s.list_a[k], at = pages_for(s.n_a[lo], q.page_size) + k - s.n_b[lo];
      q.table[(long long)seqs[lo] * q.max_pages + at] = page;
      q.refcount[page] = 1;
    }
  }
  for (int i = threadIdx.x; i < n; i += kPlan)
    if (s.n_c[i]) q.length[seqs[i]] = go ? max(s.n_a[i], new_length[i]) : s.n_a[i];
  if (threadIdx.x == 0 && status) *status = go ? 0 : bad ? bad : (int)CAB_PAGED_NO_ROOM;
}

// ------------------------------------------------------------------------------------------------ fork
// n_a: length of the parent, n_b: the fresh page of child i (-1: none), n_c: its mark was set.
__global__ void __launch_bounds__(kPlan) mla_pages_plan_fork_kernel(Pool q, const int* src, const int* dst, int n, Scratch s,
                                                                    int* status) {
  cab::after_predecessor();
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const long long most = (long long)q.max_pages * q.page_size;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    s.n_c[i] = 0;
    s.n_a[i] = 0;
    if ((unsigned)src[i] >= (unsigned)q.slots || (unsigned)dst[i] >= (unsigned)q.slots) {
      atomicMax(&bad, (int)CAB_PAGED_BAD_INDEX);
      continue;
    }
    const int len = q.length[src[i]];
    if (len < 0 || len > most) atomicMax(&bad, (int)CAB_PAGED_BAD_INDEX);
    s.n_a[i] = min(max(len, 0), (int)min(most, (long long)0x7fffffff));
  }
  __syncthreads();
  // Every entry that a child takes over, a warp per parent; one that follows itself in the list is looked at once. A page that
  // counts as free could be taken as a child's own below.
  for (int i = threadIdx.x >> 5; i < n && !bad; i += kPlan / 32) {
    if (i > 0 && src[i] == src[i - 1]) continue;
    const int need = pages_for(s.n_a[i], q.page_size);
    const int* row = q.table + (long long)src[i] * q.max_pages;
    bool lost = false;
#pragma unroll 4
    for (int k = threadIdx.x & 31; k < need; k += 32) {
      const int page = row[k];
      lost |= (unsigned)page >= (unsigned)q.num_pages || q.refcount[page] <= 0;
    }
    if (lost) atomicMax(&bad, (int)CAB_PAGED_BAD_PAGE);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n && !bad; i += kPlan) {
    const int old = atomicExch(q.length + dst[i], -1);
    if (old == -1) { atomicMax(&bad, (int)CAB_PAGED_BAD_INDEX); continue; }
    s.n_c[i] = 1;
    s.n_b[i] = old;
    if (old != 0) atomicMax(&bad, (int)CAB_PAGED_NOT_EMPTY);
  }
  __syncthreads();
  int want = 0;
  bool room = true;
  if (!bad) {
    for (int base = 0; base < n; base += kPlan) {
      const int i = base + threadIdx.x;
      int total;
      const int part = i < n && s.n_a[i] % q.page_size != 0;
      const int at = want + plan_scan(part, total);
      if (i < n) s.n_b[i] = part ? at : -1;
      want += total;
    }
    room = want <= q.num_pages && lowest_free(q.refcount, q.num_pages, want, s.list_a);
    __syncthreads();
  }
  const bool go = !bad && room;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    if (!s.n_c[i]) continue;
    if (!go) { q.length[dst[i]] = bad ? s.n_b[i] : 0; continue; }
    q.length[dst[i]] = s.n_a[i];
    const int k = s.n_b[i];
    if (k < 0) continue;
    const int last = s.n_a[i] / q.page_size, fresh = s.list_a[k];
    s.list_b[k] = q.table[(long long)src[i] * q.max_pages + last];
    q.table[(long long)dst[i] * q.max_pages + last] = fresh;
    q.refcount[fresh] = 1;
  }
  if (threadIdx.x == 0) {
    s.head[0] = go ? want : 0;
    s.head[1] = go;
    if (status) *status = go ? 0 : bad ? bad : (int)CAB_PAGED_NO_ROOM;
  }
}

// Shared pages of every child, then the data of the partly filled ones.
template <typename Unit>
__global__ void __launch_bounds__(kCopy) mla_pages_fork_kernel(Pool q, const int* src, const int* dst, int n, Scratch s,
                                                               uint8_t* pages, long long layer_stride, int layers,
                                                               long long page_bytes) {
  cab::after_predecessor();
  if (!s.head[1]) return;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int full = s.n_a[i] / q.page_size;
    const int* from = q.table + (long long)src[i] * q.max_pages;
    int* to = q.table + (long long)dst[i] * q.max_pages;
    for (int k = threadIdx.x; k < full; k += kCopy) {
      const int page = from[k];
      to[k] = page;
      if ((unsigned)page < (unsigned)q.num_pages) atomicAdd(q.refcount + page, 1);   // (the plan found it so)
    }
  }
  copy_pages<Unit>(pages, layer_stride, layers, page_bytes, s.head[0], s.list_b, s.list_a);
}

// ------------------------------------------------------------------------------------------------ free
// One CTA per listed sequence; whoever takes the length out of the array gives its pages back.
__global__ void __launch_bounds__(256) mla_pages_free_kernel(Pool q, const int* seqs, int n, int* status) {
  cab::after_predecessor();
  __shared__ int taken;
  const int seq = seqs[blockIdx.x];
  if ((unsigned)seq >= (unsigned)q.slots) {
    if (threadIdx.x == 0) raise(status, CAB_PAGED_BAD_INDEX);
    return;
  }
  if (threadIdx.x == 0) taken = atomicExch(q.length + seq, 0);
  __syncthreads();
  const int need = min(pages_for(max(taken, 0), q.page_size), q.max_pages);
  int* row = q.table + (long long)seq * q.max_pages;
  for (int k = threadIdx.x; k < need; k += 256) {
    const int page = row[k];
    row[k] = -1;
    if ((unsigned)page >= (unsigned)q.num_pages) { raise(status, CAB_PAGED_BAD_PAGE); continue; }
    if (atomicSub(q.refcount + page, 1) <= 0) {          // was free already: the table and the counts disagree
      atomicAdd(q.refcount + page, 1);
      raise(status, CAB_PAGED_BAD_PAGE);
    }
  }
}

// ------------------------------------------------------------------------------------------------ compact
// list_b -> list_a: the moves; map[p]: where page p went, p itself if it stayed, -1 if it was free.
__global__ void __launch_bounds__(kPlan) mla_pages_plan_compact_kernel(int* refcount, int num_pages, Scratch s, int* status) {
  cab::after_predecessor();
  if (threadIdx.x == 0 && status) *status = 0;
  int used = 0;
  for (int base = 0; base < num_pages; base += kPlan * kScan) {
    const int p0 = base + threadIdx.x * kScan;
    int mine = 0, total;
#pragma unroll
    for (int k = 0; k < kScan; ++k) mine += p0 + k < num_pages && refcount[p0 + k] > 0;
    plan_scan(mine, total);
    used += total;
  }
  int holes = 0, high = 0;                     // free pages below U and used ones from U on: as many of either
  for (int base = 0; base < num_pages; base += kPlan * kScan) {
    const int p0 = base + threadIdx.x * kScan;
    bool hole[kScan], move[kScan];
    int a = 0, b = 0, total;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      const int p = p0 + k;
      const bool in = p < num_pages, is = in && refcount[p] > 0;
      hole[k] = in && !is && p < used;
      move[k] = is && p >= used;
      a += hole[k];
      b += move[k];
    }
    int at = holes + plan_scan(a, total);
    holes += total;
#pragma unroll
    for (int k = 0; k < kScan; ++k)
      if (hole[k]) s.list_a[at++] = p0 + k;
    at = high + plan_scan(b, total);
    high += total;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      const int p = p0 + k;
      if (p < num_pages) s.map[p] = move[k] ? at : p < used && !hole[k] ? p : -1;
      if (move[k]) s.list_b[at++] = p;
    }
  }
  __syncthreads();
  for (int p = used + threadIdx.x; p < num_pages; p += kPlan)
    if (s.map[p] >= 0) s.map[p] = s.list_a[s.map[p]];
  __syncthreads();
  for (int k = threadIdx.x; k < high; k += kPlan) {
    refcount[s.list_a[k]] = refcount[s.list_b[k]];
    refcount[s.list_b[k]] = 0;
  }
  if (threadIdx.x == 0) s.head[0] = high;
}

template <typename Unit>
__global__ void __launch_bounds__(kCopy) mla_pages_compact_kernel(Pool q, Scratch s, uint8_t* pages, long long layer_stride,
                                                                  int layers, long long page_bytes, int* status) {
  cab::after_predecessor();
  for (int seq = blockIdx.x; seq < q.slots; seq += gridDim.x) {
    const int need = min(pages_for(max(q.length[seq], 0), q.page_size), q.max_pages);
    int* row = q.table + (long long)seq * q.max_pages;
    for (int k = threadIdx.x; k < need; k += kCopy) {
      const int page = row[k];
      if ((unsigned)page >= (unsigned)q.num_pages) { raise(status, CAB_PAGED_BAD_PAGE); continue; }
      const int to = s.map[page];
      if (to < 0) raise(status, CAB_PAGED_BAD_PAGE);
      else if (to != page) row[k] = to;
    }
  }
  copy_pages<Unit>(pages, layer_stride, layers, page_bytes, s.head[0], s.list_b, s.list_a);
}

// Widest access that every page start allows.
int unit_of(const void* pages, long long layer_stride, long long page_bytes) {
  const unsigned long long all = reinterpret_cast<unsigned long long>(pages) | (unsigned long long)layer_stride |
                                 (unsigned long long)page_bytes;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
}
// CTAs of the launch that moves `moves` pages and walks `rows` table rows: no more than the work, eight an SM.
unsigned grid_of(long long moves, int layers, long long page_bytes, int unit, long long rows) {
  const long long pieces = (page_bytes / unit + 4 * kCopy - 1) / (4 * kCopy);
  const long long work = moves * layers * pieces;
  long long g = work > rows ? work : rows;
  if (g > 8LL * cab::kNumSMs) g = 8LL * cab::kNumSMs;
  return (unsigned)(g < 1 ? 1 : g);
}

bool bad_pool(const int* table, const int* length, const int* refcount, int slots, int max_pages, int num_pages, int page_size) {
  return !table || !length || !refcount || slots <= 0 || max_pages <= 0 || num_pages <= 0 || page_size <= 0;
}
bool bad_pages(const void* pages, long long layer_stride, int layers, long long page_bytes, int num_pages) {
  return layers < 0 || (layers > 0 && (!pages || page_bytes <= 0 || (layers > 1 && layer_stride < page_bytes * num_pages)));
}
constexpr int kMaxList = 1 << 20, kMaxPages = 1 << 28;

}  // namespace

extern "C" size_t mla_pages_scratch_bytes(int num_pages, int n) {
  if (num_pages <= 0 || n < 0) return 0;
  return (scratch_ints(num_pages, n) * 4 + 15) & ~(size_t)15;
}

// Calls LAUNCH with the type of the widest access the pages allow.
#define CAB_BY_UNIT(unit, LAUNCH)                 \
  do {                                            \
    if ((unit) == 16) { LAUNCH(uint4); }          \
    else if ((unit) == 4) { LAUNCH(uint32_t); }   \
    else { LAUNCH(uint8_t); }                     \
  } while (0)

extern "C" int mla_pages_copy_launcher(void* pages, long long layer_stride, int layers, int num_pages, long long page_bytes,
                                       const int* src, const int* dst, int n, void* scratch, int* status, int config,
                                       cudaStream_t stream) {
  (void)config;
  if (n < 0 || num_pages <= 0 || bad_pages(pages, layer_stride, layers, page_bytes, num_pages)) return CAB_ERR_BAD_ARGUMENT;
  if (n == 0 || layers == 0) {
    if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
    return CAB_OK;
  }
  if (!src || !dst || !scratch) return CAB_ERR_BAD_ARGUMENT;
  if (n > kMaxList || num_pages > kMaxPages) return CAB_ERR_TOO_LARGE;
  if (!cab::aligned_to(scratch, 16)) return CAB_ERR_MISALIGNED;
  const Scratch s = carve(scratch, num_pages, n);
  const int rc = cab::launch_behind(&mla_pages_check_copy_kernel, dim3(1), dim3(kPlan), 0, stream, src, dst, n, num_pages, s, status);
  if (rc != CAB_OK) return rc;
  const int unit = unit_of(pages, layers > 1 ? layer_stride : 0, page_bytes);
  const unsigned grid = grid_of(n, layers, page_bytes, unit, 0);
#define CAB_LAUNCH(U)                                                                                             \
  return cab::launch_behind(&mla_pages_copy_kernel<U>, dim3(grid), dim3(kCopy), 0, stream, static_cast<uint8_t*>(pages), \
                            layer_stride, layers, page_bytes, s.head, s.n_a, s.n_b)
  CAB_BY_UNIT(unit, CAB_LAUNCH);
#undef CAB_LAUNCH
}

extern "C" int mla_pages_extend_launcher(int* page_table, int* length, int* refcount, int slots, int max_pages, int num_pages,
                                         int page_size, const int* seqs, const int* new_length, int n, void* scratch,
                                         int* status, int config, cudaStream_t stream) {
  (void)config;
  if (n < 0 || bad_pool(page_table, length, refcount, slots, max_pages, num_pages, page_size)) return CAB_ERR_BAD_ARGUMENT;
  if (n == 0) {
    if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
    return CAB_OK;
  }
  if (!seqs || !new_length || !scratch) return CAB_ERR_BAD_ARGUMENT;
  if (n > kMaxList || num_pages > kMaxPages) return CAB_ERR_TOO_LARGE;
  if (!cab::aligned_to(scratch, 16)) return CAB_ERR_MISALIGNED;
  const Pool q{page_table, length, refcount, slots, max_pages, num_pages, page_size};
  return cab::launch_behind(&mla_pages_extend_kernel, dim3(1), dim3(kPlan), 0, stream, q, seqs, new_length, n,
                            carve(scratch, num_pages, n), status);
}

extern "C" int mla_pages_fork_launcher(void* pages, long long layer_stride, int layers, long long page_bytes, int* page_table,
                                       int* length, int* refcount, int slots, int max_pages, int num_pages, int page_size,
                                       const int* src, const int* dst, int n, void* scratch, int* status, int config,
                                       cudaStream_t stream) {
  (void)config;
  if (n < 0 || bad_pool(page_table, length, refcount, slots, max_pages, num_pages, page_size) ||
      bad_pages(pages, layer_stride, layers, page_bytes, num_pages))
    return CAB_ERR_BAD_ARGUMENT;
  if (n == 0) {
    if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
    return CAB_OK;
  }
  if (!src || !dst || !scratch) return CAB_ERR_BAD_ARGUMENT;
  if (n > kMaxList || num_pages > kMaxPages) return CAB_ERR_TOO_LARGE;
  if (!cab::aligned_to(scratch, 16)) return CAB_ERR_MISALIGNED;
  const Pool q{page_table, length, refcount, slots, max_pages, num_pages, page_size};
  const Scratch s = carve(scratch, num_pages, n);
  const int rc = cab::launch_behind(&mla_pages_plan_fork_kernel, dim3(1), dim3(kPlan), 0, stream, q, src, dst, n, s, status);
  if (rc != CAB_OK) return rc;
  if (layers == 0) page_bytes = 0;
  const int unit = unit_of(pages, layers > 1 ? layer_stride : 0, page_bytes);
  const unsigned grid = grid_of(n, layers, page_bytes, unit, n);
#define CAB_LAUNCH(U)                                                                                                  \
  return cab::launch_behind(&mla_pages_fork_kernel<U>, dim3(grid), dim3(kCopy), 0, stream, q, src, dst, n, s,             \
                            static_cast<uint8_t*>(pages), layer_stride, layers, page_bytes)
  CAB_BY_UNIT(unit, CAB_LAUNCH);
#undef CAB_LAUNCH
}

extern "C" int mla_pages_free_launcher(int* page_table, int* length, int* refcount, int slots, int max_pages, int num_pages,
                                       int page_size, const int* seqs, int n, int* status, int config, cudaStream_t stream) {
  (void)config;
  if (n < 0 || bad_pool(page_table, length, refcount, slots, max_pages, num_pages, page_size)) return CAB_ERR_BAD_ARGUMENT;
  if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
  if (n == 0) return CAB_OK;
  if (!seqs) return CAB_ERR_BAD_ARGUMENT;
  if (n > kMaxList || num_pages > kMaxPages) return CAB_ERR_TOO_LARGE;
  const Pool q{page_table, length, refcount, slots, max_pages, num_pages, page_size};
  return cab::launch_behind(&mla_pages_free_kernel, dim3(n), dim3(256), 0, stream, q, seqs, n, status);
}

extern "C" int mla_pages_compact_launcher(void* pages, long long layer_stride, int layers, long long page_bytes, int* page_table,
                                          const int* length, int* refcount, int slots, int max_pages, int num_pages,
                                          int page_size, void* scratch, int* status, int config, cudaStream_t stream) {
  (void)config;
  if (bad_pool(page_table, length, refcount, slots, max_pages, num_pages, page_size) ||
      bad_pages(pages, layer_stride, layers, page_bytes, num_pages) || !scratch)
    return CAB_ERR_BAD_ARGUMENT;
  if (num_pages > kMaxPages) return CAB_ERR_TOO_LARGE;
  if (!cab::aligned_to(scratch, 16)) return CAB_ERR_MISALIGNED;
  const Pool q{page_table, const_cast<int*>(length), refcount, slots, max_pages, num_pages, page_size};
  const Scratch s = carve(scratch, num_pages, 0);
  const int rc = cab::launch_behind(&mla_pages_plan_compact_kernel, dim3(1), dim3(kPlan), 0, stream, refcount, num_pages, s, status);
  if (rc != CAB_OK) return rc;
  if (layers == 0) page_bytes = 0;
  const int unit = unit_of(pages, layers > 1 ? layer_stride : 0, page_bytes);
  const unsigned grid = grid_of(num_pages / 2 + 1, layers, page_bytes, unit, slots);
#define CAB_LAUNCH(U)                                                                                           \
  return cab::launch_behind(&mla_pages_compact_kernel<U>, dim3(grid), dim3(kCopy), 0, stream, q, s,                \
                            static_cast<uint8_t*>(pages), layer_stride, layers, page_bytes, status)
  CAB_BY_UNIT(unit, CAB_LAUNCH);
#undef CAB_LAUNCH
}
