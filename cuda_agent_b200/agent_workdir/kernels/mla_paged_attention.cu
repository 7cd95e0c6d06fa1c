// Dense latent attention of each sequence's new tokens over its rows of a paged cache:
//   s_j = scale * q . c_j (576 columns),  out = sum_j softmax(s)_j c_j[:512],  lse = log sum_j exp(s_j)
// over the rows that the token may see (causal, window, length). All heads read the same rows, so the (token,
// head) pairs of a sequence are the rows of one matrix, and 128 of them make a tile whatever the head count:
// one token with 128 heads, eight tokens with 16, or a decode step's 16 rows in a tile that is mostly empty.
//
// A tile of 128 rows times 512 value columns of fp32 would take all of tensor memory, so a cluster of two CTAs shares
// a tile. Each accumulates 256 of the value columns over all keys, and forms the scores of every other 64 keys over all
// 576 columns: a step of 128 keys is 64 for either CTA. What crosses between them is P, 16 KB a step and direction.
// (Without the exchange, each CTA forming all scores for itself, the tensor core has 832 column steps a key to do
// instead of 544: 4800 clk for 128 keys, where this takes 3150, and 2730 us for the chunk below.)
//   tensor memory  O 256 columns, S 64, 192 for 384 columns of Q as the A operand: this CTA's value half, the rotary
//                  columns and 64 of the other half
//   shared memory  the other 192 columns of Q (48 KB); of the own keys the other value half in two units of 128
//                  columns (16 KB each), the rotary columns (8 KB) and the own value half (32 KB, two slots); of the
//                  other CTA's keys the own value half (32 KB); P of either CTA's keys (16 KB each)
//   tensor core    Q.K^T of step j+1, P.V of step j with the own keys, P.V with the other CTA's. So the softmax of
//                  step j has the time of a Q.K^T, and every slot is asked for again 1500 clk or more before it is
//                  read: a row comes from either die's L2, 1000 to 1500 clk away
// What bounds a step is shared memory: operands 216 KB, loads 104 KB, P 48 KB are 2940 clk at 128 bytes a clk, of 3150;
// the tensor core alone would take 2050.
// P goes to shared memory, where the tensor core reads it and a bulk copy takes it to the other CTA. (Written there by
// the threads it arrived 2000 clk later: stores to another CTA of 16 bytes a row are slow, and so are the fences.)
// A tile's first scores begin with the columns of Q in shared memory, while the others are on their way to tensor memory.
// Both CTAs must weigh a row's keys against one reference m, or their parts of O would not add up. m is a whole
// number (log2 units) that moves only in a tile's first step and when a score exceeds it by more than kJump, so P is
// computed against the m of the step before while a flag from either CTA travels: only if one says so do the two
// exchange their rows' maxima, move m, rescale O and compute P again.
//   warps 0-3  one (token, head) row per thread: softmax, exchange, result
//   warp 4     issues the tensor instructions
//   warps 5, 7 TMA: 5 for the other value half, 7 for the rest, one box per run of rows that lie in one page. Q comes
//              the same way, its tensor-memory part through slots that its tile does not need yet
//   warp 6     clears the rows behind a sequence's end in its last step's value rows
// Whoever issues tensor or TMA instructions does so in one elected thread, waits included: the operands then sit
// in uniform registers, and a wait polled by 32 lanes costs some 300 clk more than one polled by a single lane. A
// TMA instruction takes its thread 65 clk, whatever its box. A wait that is over already still costs 150 to 200 clk
// while the tensor core keeps shared memory busy, so what is loaded together lands on one barrier.
// The work of a call (tiles x steps of 128 rows) is cut into equal runs, one for each pair of CTAs, wherever
// that cuts a tile; each CTA finds its run itself from q_start and kv_len. Tiles cut by a boundary leave
// unnormalised fp32 sums, and mla_paged_merge_kernel joins them in a fixed order.
// Every wait is bounded.
// Measured, 128 heads, bf16, pages of 64: 1024 tokens after 7168 rows 1.70 ms after a rest (1289 TFLOP/s), 1.93 ms in a long
// run at the power limit (1.6 GHz); 64 sequences of 8192 rows and less, one token each, 117 and 130 us (3 TB/s of the
// cache: a step waits for its rows, the merge is 13 us of it). 32 sequences of 4096 rows and less, 5 tokens with 24
// heads, pages of 16: 49 us. One token with 16 heads and 1000 rows: 15 to 17 us, set-up and latency.
#include <cuda_fp16.h>

#include <type_traits>

#include "cab_common.cuh"
#include "sm100_primitives.cuh"

namespace {

constexpr int kD = 576, kDv = 512, kHalf = 256;
constexpr int kRows = 128;                     // (token, head) rows per tile
constexpr int kKeys = 64;                      // cache rows of a CTA in a step
constexpr int kStep = 2 * kKeys;               // and of both
constexpr int kTile = kKeys * 128;             // 64 cache rows x 64 columns, 128-byte swizzle
// 64-column tiles: units of the other value half, own value half
constexpr int kNTiles = 2, kNUnits = 2, kVTiles = 4;
// of Q: in shared memory (all of the other value half but its last), in tensor memory (own value half, rotary, that last)
constexpr int kQTiles = kNTiles * kNUnits - 1, kTTiles = kVTiles + 2;
constexpr int kVSlots = 2;
constexpr int kQChunk = kRows * 128;
constexpr int kThreads = 8 * 32;
constexpr int kQBox = 16;                      // rows of the small box for Q
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 320, kTmemCols = 512;
static_assert(kColQ + kTTiles * 32 == kTmemCols, "tensor memory");
constexpr int kMaxBatch = 16384;
constexpr float kLog2e = 1.4426950408889634f;
enum { kWaitN = 211, kWaitFree, kWaitV, kWaitS, kWaitP, kWaitPv, kWaitQ, kWaitRead, kWaitPeer };

// A sequence as this call sees it: tokens [tok, tok + n), `len` cache rows, the first token at position pos.
struct Seq { int tok, n, len, pos; };
// Steps [first, first + count) of 128 cache rows that some row of tile i sees; `units` = max(count, 1) is what
// the tile counts as when the work is divided, so that a tile that sees nothing is still written.
struct Item { int row0, rows, first, count, units; };

struct __align__(16) Control {
  // n_full: the other half's rows and the rotary columns; v_full: own half's rows of the own keys (by step), t_full: of the
  // other CTA's; x_full: the other CTA's P; q_full, q_part: Q's shared and its tensor-memory part. *_land: before clearing.
  // From the other CTA: x_full, x_first (its buffer may be written: Q came through), flag_full, max_full, sum_full (by
  // lane quadrant). From both: pv_done
  uint64_t n_full, n_empty[kNUnits], r_empty, v_full[2], v_empty[kVSlots], v_land[kVSlots], t_full, t_empty, t_land, x_full, x_first,
      s_full, s_read, p_full, pv_done, q_ready, q_full, q_part, q_free, flag_full[2][4], max_full[4], sum_full[4];
  float row_max[kRows], row_sum[kRows];         // from the other CTA
  int flag[2][4];                              // [step parity][lane quadrant] from the other CTA
  long long scan[kThreads / 32], total;
  long long x0, x1, item_x;                    // this pair's run, and where its first tile begins
  int seq, tile;                               // its first tile
  Seq first_seq;
  Item first_item;
  alignas(16) int pages[2][2][2][kKeys];       // [producer][step parity][own / other keys]: the pages of the boxes
  uint32_t tmem_base;
  int abort_flag, settled, wrong;              // wrong: the starts are not sound, nothing is computed
};
constexpr int kRingBytes = (kNUnits * kNTiles + 1 + (kVSlots + 1) * kVTiles) * kTile;
constexpr int kPBytes = kRows * 128;           // P of a CTA: 128 rows x 64 keys
constexpr int kSmemBytes = kQTiles * kQChunk + kRingBytes + 2 * kPBytes + (int)sizeof(Control) + 1024;
static_assert(kSmemBytes <= 232448 && (kMaxBatch + 2) * 4 <= kRingBytes, "shared memory");

// What the merge kernel has to know of the tile that a pair ends: its first (token, head) row, its rows, and the pair
// that holds its first part.
struct Meta { int row0, rows, first; };

struct Params {
  const void* q;
  void* out;
  float* lse;
  const int *page_table, *q_start, *kv_len;
  int T, H, batch, max_pages, num_pages, page_size;
  int box, box_log2;                           // rows of a TMA box, all in one page
  int step_pages, step_rows;                   // a step further = so many pages and rows
  uint32_t tile_bytes;                         // from one 64-column tile of a part to the next: 8192, or 1024 where the
                                               // tiles of eight rows lie after one another
  int tail;                                    // write the tokens behind the last sequence as such that see nothing
  int causal, window, rows_cap, pairs;
  float scale_log2;
  float4* part_o;                              // [pair][2][512 / 4 columns][rows_cap]: a warp writes, and the merge reads, whole lines
  float2* part_ml;                             // [pair][2][rows_cap]
  Meta* meta;                                  // [pair]
  int* status;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Issued where it stands, so that the load is under way while other work is done.
// (An ordinary load, as all of them here: the read-only path is for data that nobody writes while the kernel is there, and
// this one is there before its predecessor has ended.)
__device__ __forceinline__ int load_now(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint64_t desc_sw128(uint32_t smem_addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((smem_addr >> 4) & 0x3fff) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A commit that arrives on the same barrier of both CTAs.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(sm100::smem_u32(bar)), "h"((uint16_t)3)
               : "memory");
}
// A word for another CTA, which counts four bytes on its barrier. (An arrival with release semantics at cluster scope
// takes a thread 1100 clk here.)
__device__ __forceinline__ void send_word(uint32_t cluster_dst, uint32_t cluster_bar, uint32_t v) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
               ::"r"(cluster_dst), "r"(v), "r"(cluster_bar)
               : "memory");
}
// Copies from this CTA's shared memory to another's; the bytes count on that CTA's barrier when they are there.
__device__ __forceinline__ void bulk_copy_to(uint32_t cluster_dst, const void* src, uint32_t bytes, uint32_t cluster_bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(cluster_dst), "r"(sm100::smem_u32(src)), "r"(bytes), "r"(cluster_bar)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// One lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Cache rows as (64 columns, row of eight, column tile, eight of the page, page), in pages of less than eight rows or
// an uneven number (64 columns, row, column tile, 1, page): boxes of 1, 2 and 4 tiles; Q: boxes of 128 and 16 rows.
struct Maps { CUtensorMap one, two, four, q, q16; };

__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  const int a = min(max(p.q_start[b], 0), p.T);
  const int e = min(max(p.q_start[b + 1], a), p.T);
  s.tok = a;
  s.n = e - a;
  s.len = (int)min((long long)max(p.kv_len[b], 0), (long long)p.max_pages * p.page_size);
  s.pos = s.len - s.n;
  return s;
}
__device__ __forceinline__ int tiles_of(const Params& p, int n) {
  return (int)(((unsigned)n * (unsigned)p.H + kRows - 1) / kRows);    // T * H < 2^31
}
__device__ __forceinline__ Item item_of(const Params& p, const Seq& s, int i) {
  Item t;
  const int r0 = i * kRows, left = s.n * p.H - r0;
  t.row0 = s.tok * p.H + r0;
  t.rows = min(kRows, left);
  const int t0 = (unsigned)r0 / (unsigned)p.H, t1 = (unsigned)(r0 + t.rows - 1) / (unsigned)p.H;
  const int hi = p.causal ? min(s.len, s.pos + t1 + 1) : s.len;
  const int lo = p.window > 0 ? (int)max(0LL, (long long)s.pos + t0 + 1 - p.window) : 0;
  t.first = lo / kStep;
  t.count = hi > lo ? (hi + kStep - 1) / kStep - t.first : 0;
  t.units = max(t.count, 1);
  return t;
}

// The run of a pair as a sequence of tiles, walked in the same way by every role.
struct Walk {
  int b, i;
  long long x, x1, item_x;
  Seq s;
  Item t;
  int u0, u1;                                  // units of the tile that belong to this run
  __device__ __forceinline__ Walk(const Params& p, const Control& c)
      : b(c.seq), i(c.tile), x(c.x0), x1(c.x1), item_x(c.item_x) {
    s = c.first_seq;
    t = c.first_item;
    if (x < x1) cut();
  }
  __device__ __forceinline__ void cut() {
    u0 = (int)(x - item_x);
    u1 = (int)min((long long)t.units, x1 - item_x);
  }
  __device__ __forceinline__ bool live() const { return x < x1; }
  __device__ __forceinline__ void next(const Params& p) {
    x = item_x + u1;
    if (x >= x1) return;
    item_x += t.units;
    ++i;
    while (b < p.batch && i >= tiles_of(p, s.n)) {
      i = 0;
      if (++b < p.batch) s = seq_of(p, b);
    }
    if (b >= p.batch) { x = x1; return; }
    t = item_of(p, s, i);
    cut();
  }
  // steps of this segment, as step numbers of the sequence
  __device__ __forceinline__ int begin() const { return t.first + u0; }
  __device__ __forceinline__ int blocks() const { return t.count == 0 ? 0 : u1 - u0; }
  __device__ __forceinline__ bool whole() const { return u0 == 0 && u1 == t.units; }
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int where) {
  // one lane polls: a try_wait by 32 lanes costs some 300 clk more, which is the time of seven tensor instructions
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = sm100::mbar_wait(bar, parity, abort_flag, status, where);
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();
  return ok != 0;
}

// The same for a barrier on which the other CTA counts `bytes` (0: arrives).
__device__ __forceinline__ bool warp_wait_peer(uint64_t* bar, uint32_t parity, uint32_t bytes, volatile int* abort_flag, int* status) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) {
    if (bytes > 0) expect_bytes(sm100::smem_u32(bar), bytes);
    ok = sm100::mbar_wait_cluster(bar, parity, abort_flag, status, kWaitPeer);
  }
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();
  return ok != 0;
}

// Exclusive scan over the CTA's threads; the sum of all goes to ctl.total.
__device__ __forceinline__ long long block_scan(Control& ctl, long long v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) ctl.scan[warp] = x;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += ctl.scan[w];
    all += ctl.scan[w];
  }
  if (threadIdx.x == 0) ctl.total = all;
  __syncthreads();
  return before + x - v;
}

// The run of a pair, from what all tiles together count (W >= 1).
struct Run { int pairs; long long x0, x1; };
__device__ __forceinline__ Run run_of(long long W, int pair, int all) {
  Run r;
  r.pairs = (int)min((long long)all, W);       // no run is empty but those of the pairs behind
  if (pair >= r.pairs) { r.x0 = r.x1 = W; return r; }
  if (W < (1 << 24)) {
    r.x0 = (unsigned)W * (unsigned)pair / (unsigned)r.pairs;
    r.x1 = (unsigned)W * (unsigned)(pair + 1) / (unsigned)r.pairs;
  } else {
    r.x0 = W * pair / r.pairs;
    r.x1 = W * (pair + 1) / r.pairs;
  }
  return r;
}
// Tile i of sequence b, which begins at `at`, is where the run begins.
__device__ __forceinline__ void found(const Params& p, Control& ctl, const Run& r, long long W, int pair, long long at, int b,
                                      int i, const Seq& s, const Item& t) {
  ctl.x0 = r.x0; ctl.x1 = r.x1; ctl.item_x = at; ctl.seq = b; ctl.tile = i;
  ctl.first_seq = s;
  ctl.first_item = t;
  // the pair that ends a cut tile says so to the merge kernel
  Meta m{t.row0, 0, 0};
  if (r.x0 > at && at + t.units <= r.x1) {
    m.rows = t.rows;
    m.first = (int)(((at + 1) * r.pairs - 1) / W);             // the last pair that begins at or before `at`
  }
  if ((blockIdx.x & 1) == 0) p.meta[pair] = m;
}

// Where pair `pair` begins: thread-parallel over the sequences, then over the tiles. `pre`: batch + 1 ints of
// shared memory that nothing else uses yet. A decode step of up to 32 sequences (no more than eight tiles each) is
// settled by one warp without barriers, 1000 clk sooner. Starts that descend would give the same tokens to several
// sequences, without end, and the append writes nothing at such, at starts that begin late or that pass the tokens:
// nothing is done then.
__device__ void find_run(const Params& p, Control& ctl, int* pre, int pair) {
  const int tid = threadIdx.x;
  if (p.batch <= 32) {
    bool done = true;
    if (tid < 32) {
      Seq s{0, 0, 0, 0};
      if (tid < p.batch) s = seq_of(p, tid);
      const bool bad = __any_sync(0xffffffffu, tid < p.batch && cab::wrong_start(p.q_start, tid, p.batch, p.T));
      if (bad && tid == 0 && p.status) atomicCAS(p.status, 0, (int)CAB_PAGED_BAD_INDEX);
      const int tiles = bad ? 0 : tiles_of(p, s.n);
      done = __all_sync(0xffffffffu, tiles <= 8);
      if (done) {
        int sum = 0;
        for (int i = 0; i < tiles; ++i) sum += item_of(p, s, i).units;
        long long at = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, at, o);
          if (tid >= o) at += y;
        }
        const long long W = __shfl_sync(0xffffffffu, at, 31);
        at -= sum;
        const Run r = run_of(max(W, 1LL), pair, p.pairs);
        if (r.x0 < r.x1 && W > 0) {
          for (int i = 0; i < tiles && at <= r.x0; ++i) {
            const Item t = item_of(p, s, i);
            if (r.x0 < at + t.units) found(p, ctl, r, W, pair, at, tid, i, s, t);
            at += t.units;
          }
        } else if (tid == 0) {
          ctl.x0 = ctl.x1 = 0;
          if ((blockIdx.x & 1) == 0) p.meta[pair] = Meta{0, 0, 0};
        }
      }
      if (tid == 0) {
        ctl.settled = done;
        ctl.wrong = bad;
      }
    }
    __syncthreads();
    if (ctl.settled) return;
  }
  {
    const int per = (p.batch + kThreads - 1) / kThreads, b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    long long sum = 0;
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
      bad |= cab::wrong_start(p.q_start, b, p.batch, p.T);
      sum += tiles_of(p, seq_of(p, b).n);
    }
    bad = __syncthreads_or(bad);
    if (bad && tid == 0 && p.status) atomicCAS(p.status, 0, (int)CAB_PAGED_BAD_INDEX);
    if (tid == 0) ctl.wrong = bad;
    long long at = block_scan(ctl, bad ? 0 : sum);
    for (int b = b0; b < b1; ++b) {
      pre[b] = (int)min(at, (long long)0x7fffffff);
      at += tiles_of(p, seq_of(p, b).n);
    }
  }
  const int tiles = (int)min(ctl.total, (long long)0x7fffffff);
  if (tid == 0) pre[p.batch] = tiles;
  if (tid == 0) ctl.x0 = ctl.x1 = 0;
  __syncthreads();
  const int per = (tiles + kThreads - 1) / kThreads;
  const int i0 = (int)min((long long)tid * per, (long long)tiles), i1 = min(i0 + per, tiles);
  int b = 0;
  if (i0 < i1) {                               // last b with pre[b] <= i0
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= i0) lo = mid; else hi = mid;
    }
    b = lo;
  }
  long long sum = 0;
  if (i0 < i1) {
    int bb = b;
    Seq s = seq_of(p, bb);
    for (int i = i0; i < i1; ++i) {
      while (pre[bb + 1] <= i) s = seq_of(p, ++bb);
      sum += item_of(p, s, i - pre[bb]).units;
    }
  }
  long long at = block_scan(ctl, sum);
  const long long W = ctl.total;
  const Run r = run_of(max(W, 1LL), pair, p.pairs);
  if (W > 0 && r.x0 < r.x1 && at <= r.x0 && r.x0 < at + sum) {
    Seq s = seq_of(p, b);
    for (int i = i0; i < i1; ++i) {
      while (pre[b + 1] <= i) s = seq_of(p, ++b);
      const Item t = item_of(p, s, i - pre[b]);
      if (r.x0 < at + t.units) {
        found(p, ctl, r, W, pair, at, b, i - pre[b], s, t);
        break;
      }
      at += t.units;
    }
  }
  if ((W == 0 || r.x0 >= r.x1) && tid == 0 && (blockIdx.x & 1) == 0) p.meta[pair] = Meta{0, 0, 0};
  __syncthreads();
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
mla_paged_attention_kernel(const Params p, const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = base;
  uint8_t* n_ring = base + kQTiles * kQChunk;
  uint8_t* r_tile = n_ring + kNUnits * kNTiles * kTile;
  uint8_t* v_ring = r_tile + kTile;
  uint8_t* t_tiles = v_ring + kVSlots * kVTiles * kTile;
  uint8_t* x_tile = t_tiles + kVTiles * kTile;
  uint8_t* p_tile = x_tile + kPBytes;
  Control& ctl = *reinterpret_cast<Control*>(p_tile + kPBytes);
  // the same in all lanes, and known to be: the tensor instructions take their operands from uniform registers
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int half = blockIdx.x & 1, pair = blockIdx.x >> 1;     // half: the rank in the cluster

  if (threadIdx.x == 0) {
    sm100::mbar_init(&ctl.n_full, kNUnits + 1);
    for (int s = 0; s < kNUnits; ++s) sm100::mbar_init(&ctl.n_empty[s], 1);
    sm100::mbar_init(&ctl.r_empty, 1);
    for (int s = 0; s < 2; ++s) sm100::mbar_init(&ctl.v_full[s], 1);
    for (int s = 0; s < kVSlots; ++s) { sm100::mbar_init(&ctl.v_empty[s], 1); sm100::mbar_init(&ctl.v_land[s], 1); }
    for (uint64_t* b : {&ctl.t_full, &ctl.t_empty, &ctl.t_land, &ctl.x_full, &ctl.x_first, &ctl.s_full, &ctl.q_full, &ctl.q_part,
                        &ctl.q_free})
      sm100::mbar_init(b, 1);
    sm100::mbar_init(&ctl.pv_done, 2);
    for (uint64_t* b : {&ctl.s_read, &ctl.p_full, &ctl.q_ready}) sm100::mbar_init(b, 4);
    for (int s = 0; s < 4; ++s)
      for (uint64_t* b : {&ctl.flag_full[0][s], &ctl.flag_full[1][s], &ctl.max_full[s], &ctl.sum_full[s]}) sm100::mbar_init(b, 1);
    ctl.abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (warp == 4) {
    sm100::tmem_alloc(&ctl.tmem_base, kTmemCols);
    sm100::tmem_relinquish();
  }
  if (warp == 5 && lane == 0) {
    for (const CUtensorMap* m : {&maps.one, &maps.two, &maps.four, &maps.q, &maps.q16}) sm100::prefetch_tensormap(m);
  }
  cudaGridDependencySynchronize();             // up to here nothing of what earlier work wrote was read
  find_run(p, ctl, reinterpret_cast<int*>(n_ring), pair);
  sm100::fence_proxy_async();                  // the rings were used as scratch
  sm100::tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();                            // both CTAs' barriers exist before anything of the other's arrives on them
  if (warp <= 4) cluster_wait();
  sm100::tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl.tmem_base, 0);
  volatile int* abort_flag = &ctl.abort_flag;
  constexpr uint32_t kFmt = std::is_same_v<T, __half> ? 0 : 1;

  if (warp == 5 || warp == 7) {
    // ---------------------------------------------------------------- loads
    const int ring = warp == 7;                // 0: the other value half; 1: rotary columns, own value half of all keys
    const int other = half ? 0 : 4;            // first of the four column tiles of the other value half
    uint32_t g = 0, seg = 0, v_at = 0, t_at = 0;               // steps, segments, slots of V and uses of T (with Q) so far
    uint32_t v_landed[kVSlots] = {}, t_landed = 0;
    bool ok = true;
    const uint32_t n_base = sm100::smem_u32(n_ring), v_base = sm100::smem_u32(v_ring), t_base = sm100::smem_u32(t_tiles);
    // Entries lane + 32 k of a list of pages: 64 for the own keys' boxes, 64 for the other CTA's. Where they begin,
    // counted from the step's first row.
    int at_pages[4], at_rows[4], next[4], first_page = 0, first_row = 0;
    auto offset = [&](int k) {                 // in the step; -1: no such box
      const int e = lane + 32 * k, box = (e & 63) << p.box_log2;
      return box < kKeys ? ((e < 64) == (half == 0) ? 0 : kKeys) + box : -1;
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned off = max(offset(k), 0);
      at_pages[k] = off / (unsigned)p.page_size;
      at_rows[k] = off % (unsigned)p.page_size;
    }
    auto look = [&](const Walk& w, int j) {    // asks for the pages of step j
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k >= 2 && ring == 0) break;
        const int off = offset(k), at = first_page + at_pages[k] + (first_row + at_rows[k] >= p.page_size);
        if (off >= 0 && j * kStep + off < w.s.len) next[k] = load_now(p.page_table + (size_t)w.b * p.max_pages + at);
        else next[k] = 0;
      }
    };
    auto step = [&]() {                        // to the next step
      first_page += p.step_pages;
      first_row += p.step_rows;
      if (first_row >= p.page_size) { first_row -= p.page_size; ++first_page; }
    };
    auto keep = [&](uint32_t parity) {         // one outside the pool: TMA fills with zeros
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k >= 2 && ring == 0) break;
        if ((unsigned)next[k] >= (unsigned)p.num_pages) {
          if (p.status) atomicCAS(p.status, 0, (int)CAB_PAGED_BAD_PAGE);
          next[k] = p.num_pages;
        }
        if (k % 2 == 0 || p.box == 1) ctl.pages[ring][parity][k >> 1][lane + 32 * (k & 1)] = next[k];
      }
      __syncwarp();
    };
    // a slot of a ring, free again for its use number `at`
    auto room = [&](uint64_t* empty, uint32_t slots, uint32_t at) {
      return at < slots || sm100::mbar_wait(empty + at % slots, (at / slots - 1) & 1, abort_flag, p.status, kWaitFree);
    };
    // Rows [0, min(64, left)) of a CTA's keys, `tiles` column tiles from `from` on, in boxes that begin at row `row` of page
    // list[0]
    auto part = [&](uint32_t dst, uint32_t bar, int from, int tiles, int left, int row, const int* list) {
      const int boxes = left > 0 ? (min(kKeys, left) + p.box - 1) >> p.box_log2 : 0;
      expect_bytes(bar, tiles * boxes * p.box * 128);
      const CUtensorMap* map = p.box < 8 || tiles == 1 ? &maps.one : tiles == 2 ? &maps.two : &maps.four;
      // one copy of the instruction, in loops: unrolled over eight boxes it took 1500 clk a part, for two boxes as for eight
      const int rounds = p.box < 8 ? tiles : 1, bytes = (p.box < 8 ? 1 : tiles) * p.box * 128;
#pragma unroll 1
      for (int c = 0; c < rounds; ++c) {
        int r = row;
#pragma unroll 1
        for (int e = 0; e < boxes; ++e) {
          tma_load_5d(dst + c * kTile + e * bytes, map, bar, p.box < 8 ? r : 0, from + c, p.box < 8 ? 0 : r >> 3, list[e]);
          r += p.box;
          if (r == p.page_size) r = 0;
        }
      }
    };
    for (Walk w(p, ctl); w.live() && ok; w.next(p)) {
      const int nb = w.blocks();
      if (nb == 0) continue;
      first_page = (unsigned)(w.begin() * kStep) / (unsigned)p.page_size;
      first_row = (unsigned)(w.begin() * kStep) % (unsigned)p.page_size;
      int own_row = (unsigned)(first_row + half * kKeys) % (unsigned)p.page_size;
      int their_row = (unsigned)(first_row + (half ^ 1) * kKeys) % (unsigned)p.page_size;
      auto further = [&](int row) {
        row += p.step_rows;
        return row >= p.page_size ? row - p.page_size : row;
      };
      look(w, w.begin());
      if (elect_one()) {                       // Q of this tile
        const bool many = w.t.rows > 4 * kQBox;
        const int boxes = many ? 1 : (w.t.rows + kQBox - 1) / kQBox, rows = many ? kRows : kQBox;
        const CUtensorMap* map = many ? &maps.q : &maps.q16;
        // ring 0: its tiles of Q to where they stay. Ring 1: two tiles through T, two through a slot of V, one through
        // either buffer for P (free when T is, and when the other CTA has read the last P)
        if (ring == 0) ok = seg == 0 || sm100::mbar_wait(&ctl.q_free, (seg - 1) & 1, abort_flag, p.status, kWaitQ);
        else ok = room(ctl.v_empty, kVSlots, v_at) && room(&ctl.t_empty, 1, t_at) && room(&ctl.pv_done, 1, g);
        if (ok) {
          const uint32_t bar = sm100::smem_u32(ring == 0 ? &ctl.q_full : &ctl.q_part);
          const int tiles = ring == 0 ? kQTiles : kTTiles;
          expect_bytes(bar, tiles * boxes * rows * 128);
#pragma unroll 1
          for (int c = 0; c < tiles; ++c) {
            uint32_t dst = sm100::smem_u32(q_smem) + c * kQChunk;
            int col = 64 * (other + c);
            if (ring == 1) {
              dst = c < 2 ? t_base + c * kQChunk : c < kVTiles ? v_base + v_at % kVSlots * kVTiles * kTile + (c - 2) * kQChunk
                                                               : sm100::smem_u32(x_tile) + (c - kVTiles) * kQChunk;
              col = c < kVTiles ? 64 * (4 - other + c) : c == kVTiles ? kDv : 64 * (other + kQTiles);
            }
#pragma unroll 1
            for (int e = 0; e < boxes; ++e) tma_load_2d(dst + e * rows * 128, map, bar, col, w.t.row0 + e * rows);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++seg;
      ++v_at;
      ++t_at;
      keep(g & 1);
      // own keys of step k, then (ring 1) the other CTA's of step k - 1: in the order in which their slots become free
      for (int k = 0; k < nb + ring; ++k) {
        const int j = w.begin() + k, len = w.s.len;
        if (k < nb) step();
        if (k + 1 < nb) look(w, j + 1);
        if (elect_one()) {
          if (k < nb) {
            const int left = len - j * kStep - half * kKeys;
            const int* list = ctl.pages[ring][g & 1][0];
            const uint32_t full = sm100::smem_u32(&ctl.n_full);
            if (ring == 0) {
#pragma unroll
              for (int u = 0; u < kNUnits; ++u) {
                ok = ok && room(&ctl.n_empty[u], 1, g);
                if (ok) part(n_base + u * kNTiles * kTile, full, other + u * kNTiles, kNTiles, left, own_row, list);
              }
            } else {
              ok = room(&ctl.r_empty, 1, g);
              if (ok) {
                part(sm100::smem_u32(r_tile), full, 8, 1, left, own_row, list);
                ok = room(ctl.v_empty, kVSlots, v_at);
              }
              if (ok) {                        // rows behind the sequence's end: to the clearing warp first
                const uint32_t s = v_at % kVSlots;
                const bool tail = left < kKeys;
#pragma unroll
                for (int e = 0; e < kVSlots; ++e) v_landed[e] += tail && s == e;
                part(v_base + s * kVTiles * kTile, sm100::smem_u32(tail ? &ctl.v_land[s] : &ctl.v_full[g & 1]), 4 - other, kVTiles,
                     left, own_row, list);
              }
            }
          }
          if (ring == 1 && ok && k > 0) {
            const int left = len - (j - 1) * kStep - (half ^ 1) * kKeys;
            ok = room(&ctl.t_empty, 1, t_at);
            if (ok) {
              const bool tail = left < kKeys;
              t_landed += tail;
              part(t_base, sm100::smem_u32(tail ? &ctl.t_land : &ctl.t_full), 4 - other, kVTiles, left, their_row,
                   ctl.pages[ring][(g - 1) & 1][1]);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        own_row = further(own_row);            // of step k + 1, and the other CTA's of step k
        if (k > 0) { ++t_at; their_row = further(their_row); }
        if (k < nb) { ++g; ++v_at; }
        if (k + 1 < nb) keep(g & 1);
      }
    }
    // Giving up: nothing that is on its way may land after the CTA has ended. The last use of every slot is waited
    // for, with a limit.
    if (!ok && elect_one()) {                  // counted: what was asked for, and up to a step more
      int never = 0;
      auto drain = [&](uint64_t* bar, uint32_t uses) {
        if (uses > 0) sm100::mbar_wait_limited(bar, (uses - 1) & 1, &never, nullptr, kWaitQ, 20000000LL);
      };
      drain(&ctl.n_full, g);
      drain(&ctl.n_full, g + 1);
      if (ring == 0) {
        drain(&ctl.q_full, seg);
      } else {
        drain(&ctl.q_part, seg);
        drain(&ctl.t_full, g);
        drain(&ctl.t_land, t_landed);
        for (int e = 0; e < 2; ++e) drain(&ctl.v_full[e], (g + 2 - e) / 2);
#pragma unroll
        for (int e = 0; e < kVSlots; ++e) drain(&ctl.v_land[e], v_landed[e]);
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    // ---------------------------------------------------------------- rows behind a sequence's end
    // They may hold anything, also NaN, which a weight of zero would keep.
    uint32_t v_at = 0, g = 0, v_cleared[kVSlots] = {}, t_cleared = 0;
    bool ok = true;
    const uint32_t group = p.tile_bytes == 1024 ? kVTiles * 1024 : 1024;
    auto clear = [&](uint8_t* v, int valid) {
      for (int e = valid * 8 + lane; e < kKeys * 8; e += 32)     // 16 bytes each, 64 to eight rows
#pragma unroll
        for (int c = 0; c < kVTiles; ++c)
          *reinterpret_cast<uint4*>(v + c * p.tile_bytes + (e >> 6) * group + (e & 63) * 16) = make_uint4(0, 0, 0, 0);
      sm100::fence_proxy_async();
      __syncwarp();
    };
    for (Walk w(p, ctl); w.live() && ok; w.next(p)) {
      const int nb = w.blocks();
      if (nb == 0) continue;
      ++v_at;                                  // Q
      // only a segment's last step can be the sequence's last
      const int left = w.s.len - (w.begin() + nb - 1) * kStep;
      const int mine = left - half * kKeys, theirs = left - (half ^ 1) * kKeys;
      if (mine < kKeys) {
        const uint32_t s = (v_at + nb - 1) % kVSlots;
        uint32_t uses = 0;
#pragma unroll
        for (int e = 0; e < kVSlots; ++e)
          if (s == e) uses = v_cleared[e]++;
        if (!warp_wait(&ctl.v_land[s], uses & 1, abort_flag, p.status, kWaitV)) { ok = false; break; }
        clear(v_ring + s * kVTiles * kTile, max(mine, 0));
        if (lane == 0) sm100::mbar_arrive(&ctl.v_full[(g + nb - 1) & 1]);
      }
      if (theirs < kKeys) {
        if (!warp_wait(&ctl.t_land, t_cleared++ & 1, abort_flag, p.status, kWaitV)) { ok = false; break; }
        clear(t_tiles, max(theirs, 0));
        if (lane == 0) sm100::mbar_arrive(&ctl.t_full);
      }
      v_at += nb;
      g += nb;
    }
  } else if (warp == 4) {
    // ---------------------------------------------------------------- tensor core
    // One thread: nothing here is done by a warp together.
    if (elect_one()) {
      constexpr uint32_t idesc_qk = sm100::umma_idesc(kFmt, kRows, kKeys);
      constexpr uint32_t idesc_pv = sm100::umma_idesc(kFmt, kRows, kHalf) | (1u << 16);   // V: keys down, columns along
      // rows of a step, by what the boxes left: tiles of 8 KB, or the tiles of eight rows after one another
      const bool by_rows = p.tile_bytes == 1024;
      const uint64_t q_desc = desc_sw128(sm100::smem_u32(q_smem), 16, 1024);
      const uint64_t n_desc = desc_sw128(sm100::smem_u32(n_ring), 16, by_rows ? kNTiles * 1024 : 1024);
      const uint64_t r_desc = desc_sw128(sm100::smem_u32(r_tile), 16, 1024);
      const uint32_t v_group = by_rows ? kVTiles * 1024 : 1024, tile = p.tile_bytes >> 4;
      const uint64_t vk_desc = desc_sw128(sm100::smem_u32(v_ring), 16, v_group);
      const uint64_t vn_desc = desc_sw128(sm100::smem_u32(v_ring), p.tile_bytes, v_group);
      const uint64_t tn_desc = desc_sw128(sm100::smem_u32(t_tiles), p.tile_bytes, v_group);
      const uint64_t x_desc = desc_sw128(sm100::smem_u32(x_tile), 16, 1024), p_desc = desc_sw128(sm100::smem_u32(p_tile), 16, 1024);
      uint32_t v_qk = 0, v_pv = 0, g_qk = 0, g_pv = 0, seg = 0;
      bool ok = true;
      for (Walk w(p, ctl); w.live() && ok; w.next(p)) {
        const int nb = w.blocks();
        if (nb == 0) continue;
        if (!sm100::mbar_wait(&ctl.q_full, seg & 1, abort_flag, p.status, kWaitQ)) break;
        const uint32_t x_bytes = (w.t.rows + 31) / 32 * 32 * 128;                // what the other CTA's warps send in a step
        for (int k = 0; k <= nb; ++k) {
          if (k < nb) {                        // S = Q . K^T of step k, own keys
            if (!sm100::mbar_wait(&ctl.n_full, g_qk & 1, abort_flag, p.status, kWaitN)) { ok = false; break; }
            if (g_qk > 0 && !sm100::mbar_wait(&ctl.s_read, (g_qk - 1) & 1, abort_flag, p.status, kWaitRead)) { ok = false; break; }
            sm100::tc_fence_after_sync();
            const uint32_t d = tmem + kColS;
#pragma unroll
            for (int u = 0; u < kNUnits; ++u) {
              const uint64_t b = n_desc + u * kNTiles * (kTile >> 4);
#pragma unroll
              for (int c = 0; c < kNTiles; ++c) {
                if (u * kNTiles + c == kQTiles && k == 0) {        // the rest of Q: the parts before it did not need it
                  ok = sm100::mbar_wait(&ctl.q_ready, seg & 1, abort_flag, p.status, kWaitQ);
                  if (!ok) break;
                  ++seg;
                  sm100::mbar_arrive(&ctl.v_empty[v_qk % kVSlots]);        // where Q came through was read
                  sm100::mbar_arrive(&ctl.t_empty);
                  sm100::mbar_arrive_cluster_relaxed(sm100::cluster_map(sm100::smem_u32(&ctl.x_first), half ^ 1));
                  ++v_qk;
                  ++v_pv;
                  sm100::tc_fence_after_sync();
                }
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                  const int t = u * kNTiles + c;
                  if (t < kQTiles)
                    sm100::umma_f16(d, q_desc + t * (kQChunk >> 4) + 2 * k4, b + c * tile + 2 * k4, idesc_qk, t > 0 || k4 > 0 ? 1u : 0u);
                  else
                    umma_ts(d, tmem + kColQ + (kTTiles - 1) * 32 + k4 * 8, b + c * tile + 2 * k4, idesc_qk, 1u);
                }
              }
              if (!ok) break;
              sm100::umma_commit(&ctl.n_empty[u]);
            }
            if (!ok) break;
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4)
              umma_ts(d, tmem + kColQ + kVTiles * 32 + k4 * 8, r_desc + 2 * k4, idesc_qk, 1u);
            sm100::umma_commit(&ctl.r_empty);
            const uint32_t s = v_qk % kVSlots;
            if (!sm100::mbar_wait(&ctl.v_full[g_qk & 1], (g_qk >> 1) & 1, abort_flag, p.status, kWaitV)) { ok = false; break; }
#pragma unroll
            for (int c = 0; c < kVTiles; ++c) {
              const uint64_t b = vk_desc + s * kVTiles * (kTile >> 4) + c * tile;
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) umma_ts(d, tmem + kColQ + c * 32 + k4 * 8, b + 2 * k4, idesc_qk, 1u);
            }
            sm100::umma_commit(&ctl.s_full);
            if (k + 1 == nb) sm100::umma_commit(&ctl.q_free);
            ++g_qk;
            ++v_qk;
          }
          if (k > 0) {                         // O += P . V of step k - 1: own keys, then the other CTA's
            const uint32_t s = v_pv % kVSlots;
            expect_bytes(sm100::smem_u32(&ctl.x_full), x_bytes);                   // the last one was waited for
            if (!sm100::mbar_wait(&ctl.p_full, g_pv & 1, abort_flag, p.status, kWaitP)) { ok = false; break; }
            sm100::tc_fence_after_sync();
            const uint64_t b = vn_desc + s * kVTiles * (kTile >> 4);
#pragma unroll
            for (int k4 = 0; k4 < kKeys / 16; ++k4)
              sm100::umma_f16(tmem + kColO, p_desc + 2 * k4, b + k4 * (v_group >> 3), idesc_pv, (k > 1 || k4 > 0) ? 1u : 0u);
            sm100::umma_commit(&ctl.v_empty[s]);
            if (!sm100::mbar_wait(&ctl.t_full, g_pv & 1, abort_flag, p.status, kWaitV) ||
                !sm100::mbar_wait_cluster(&ctl.x_full, g_pv & 1, abort_flag, p.status, kWaitPeer)) { ok = false; break; }
            sm100::tc_fence_after_sync();
#pragma unroll
            for (int k4 = 0; k4 < kKeys / 16; ++k4)
              sm100::umma_f16(tmem + kColO, x_desc + 2 * k4, tn_desc + k4 * (v_group >> 3), idesc_pv, 1u);
            sm100::umma_commit(&ctl.t_empty);
            umma_commit_both(&ctl.pv_done);
            ++g_pv;
            ++v_pv;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax, one row per thread
    // Weights grow to 2^kJump before m moves, to kBias below the maximum. fp16: so high that small weights stay normal
    // numbers. bf16 has the exponents: a move costs an exchange and a pass over O, and with 8 instead of 24 there are
    // enough for 4 % of the time of a long chunk; the weighted sum of 10^5 rows stays finite for values up to 10^26.
    constexpr float kJump = std::is_same_v<T, __half> ? 15.f : 24.f, kBias = std::is_same_v<T, __half> ? 6.f : 0.f;
    const int row = threadIdx.x;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const uint32_t peer = half ^ 1;
    auto there = [&](const void* mine) { return sm100::cluster_map(sm100::smem_u32(mine), peer); };
    const uint32_t x_there = there(x_tile) + warp * 32 * 128, x_full_there = there(&ctl.x_full);
    const uint32_t flag_there = there(&ctl.flag[0][warp]), flag_full_there = there(&ctl.flag_full[0][warp]);
    const uint32_t max_there = there(&ctl.row_max[row]), max_full_there = there(&ctl.max_full[warp]);
    const uint32_t sum_there = there(&ctl.row_sum[row]), sum_full_there = there(&ctl.sum_full[warp]);
    uint32_t g = 0, v_at = 0, seg = 0;         // steps, slots of V and tiles with steps so far
    uint32_t flags = 0, moves = 0, sums = 0;   // exchanges of this warp so far
    bool ok = true;
    const int own = half * kHalf;
    // Columns of Q to tensor memory, a row per thread: two tiles of 64 columns from T, two from a slot of V, one from
    // either buffer for P.
    auto take_q = [&]() {
      if (!warp_wait(&ctl.q_part, seg & 1, abort_flag, p.status, kWaitQ)) { ok = false; return; }
      const uint8_t* slot = v_ring + v_at % kVSlots * kVTiles * kTile;
#pragma unroll 1
      for (int c = 0; c < kTTiles; ++c) {
        const uint8_t* src = (c < 2 ? t_tiles + c * kQChunk : c < kVTiles ? slot + (c - 2) * kQChunk : x_tile + (c - kVTiles) * kQChunk) + row * 128;
        uint32_t u[32];
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + ((v ^ (row & 7)) << 4));
          u[4 * v] = x.x; u[4 * v + 1] = x.y; u[4 * v + 2] = x.z; u[4 * v + 3] = x.w;
        }
        tmem_st_32x32(lanes + kColQ + c * 32, u);
      }
      ++v_at;
      ++seg;
      tmem_st_wait();
      sm100::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&ctl.q_ready);
    };

    // Q of the next tile with steps, if there is one: it goes in as soon as the last scores are out.
    auto next_q = [&](Walk n) {
      while (n.live() && n.blocks() == 0) n.next(p);
      if (n.live()) take_q();
    };
    Walk w(p, ctl);
    next_q(w);
    while (w.live() && ok) {
      const int nb = w.blocks();
      // what this row sees: cache rows [lo, hi)
      const int tok = (int)((unsigned)(w.t.row0 + row) / (unsigned)p.H) - w.s.tok;
      const bool live = row < w.t.rows;
      int hi = p.causal ? min(w.s.len, w.s.pos + tok + 1) : w.s.len;
      const int lo = p.window > 0 ? (int)max(0LL, (long long)w.s.pos + tok + 1 - p.window) : 0;
      if (!live) hi = 0;
      const bool warp_live = warp * 32 < w.t.rows;             // the same in both CTAs
      float m_ref = -INFINITY, l_sum = 0.f;
      for (int k = 0; k < nb; ++k, ++g) {
        if (!warp_wait(&ctl.s_full, g & 1, abort_flag, p.status, kWaitS)) { ok = false; break; }
        sm100::tc_fence_after_sync();
        uint32_t u0[32], u1[32], pk[32];
        if (warp_live) {
          sm100::tmem_ld_32x32(lanes + kColS, u0);
          sm100::tmem_ld_32x32(lanes + kColS + 32, u1);
          sm100::tmem_ld_wait();
        }
        sm100::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&ctl.s_read);        // the next step's scores may overwrite them
        bool moved = false;
        float factor = 1.f;
        if (warp_live) {
          const int key0 = (w.begin() + k) * kStep + half * kKeys;
          if (!__all_sync(0xffffffffu, lo <= key0 && key0 + kKeys <= hi)) {
            const unsigned a = (unsigned)(key0 - lo), span = hi > lo ? (unsigned)(hi - lo) : 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (a + i >= span) u0[i] = 0xff800000u;
              if (a + 32 + i >= span) u1[i] = 0xff800000u;
            }
          }
          float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            m0 = fmaxf(m0, __uint_as_float(u0[i]));
            m1 = fmaxf(m1, __uint_as_float(u1[i]));
          }
          const float m_own = fmaxf(m0, m1) * p.scale_log2;      // scale > 0: the maximum commutes with it
          // bit 0: m has to move, as a score exceeds it by too much or in the first step, which needs no flag. Bit 1: below, a
          // score is multiplied and m subtracted with one rounding; where the product's own rounding is a matter of whole
          // units, the largest score could end far above m, so the products are rounded first, as m was.
          const unsigned what = __reduce_or_sync(0xffffffffu, (k == 0 || m_own > m_ref + kJump ? 1u : 0u) |
                                                                  (fabsf(m_own) > 0x1p22f && m_own != -INFINITY ? 2u : 0u));
          const int jump = what & 1;
          float scale = p.scale_log2;
          if (what & 2) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              u0[i] = __float_as_uint(__uint_as_float(u0[i]) * scale);
              u1[i] = __float_as_uint(__uint_as_float(u1[i]) * scale);
            }
            scale = 1.f;
          }
          if (k > 0 && lane == 0) {
            expect_bytes(sm100::smem_u32(&ctl.flag_full[flags & 1][warp]), 4);
            send_word(flag_there + (flags & 1) * 16, flag_full_there + (flags & 1) * 32, jump);
          }
          float sum = 0.f;
          // twice at most; a loop, so that its code is there once: the first step waits for code as much as for data
#pragma unroll 1
          for (int pass = 0;; ++pass) {
            if (pass > 0 || !jump) {
              const float neg = m_ref == -INFINITY ? 0.f : -m_ref;   // masked scores: exp2(-inf) = 0
              float s0 = 0.f, s1 = 0.f;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float a = exp2_approx(fmaf(__uint_as_float(u0[i]), scale, neg));
                const float b = exp2_approx(fmaf(__uint_as_float(u0[i + 1]), scale, neg));
                const float c = exp2_approx(fmaf(__uint_as_float(u1[i]), scale, neg));
                const float d = exp2_approx(fmaf(__uint_as_float(u1[i + 1]), scale, neg));
                s0 += a + b;
                s1 += c + d;
                // P is rounded to the cache's 16-bit type, the only form the tensor core takes beside it: half a
                // step of 2^-8 (bf16) or 2^-11 (fp16) per weight, as much as the rounding of the result itself
                pk[i >> 1] = pack2<T>(a, b);
                pk[16 + (i >> 1)] = pack2<T>(c, d);
              }
              sum = s0 + s1;
              if (pass > 0) break;
            }
            if (k > 0) {                       // two barriers in turn: the other CTA may be a step ahead, not two
              int jump_there = 0, got = 1;
              if (lane == 0) {
                got = sm100::mbar_wait_cluster(&ctl.flag_full[flags & 1][warp], (flags >> 1) & 1, abort_flag, p.status, kWaitPeer);
                jump_there = *reinterpret_cast<volatile int*>(&ctl.flag[flags & 1][warp]);
              }
              jump_there = __shfl_sync(0xffffffffu, got ? jump_there : -1, 0);
              ok = jump_there >= 0;
              ++flags;
              if (!ok || !(jump | jump_there)) break;
            }
            // both CTAs' warps of these rows come here together
            send_word(max_there, max_full_there, __float_as_uint(m_own));
            ok = warp_wait_peer(&ctl.max_full[warp], moves & 1, 128, abort_flag, p.status);
            if (!ok) break;
            ++moves;
            const float top = fmaxf(m_own, *reinterpret_cast<volatile float*>(&ctl.row_max[row]));
            if (top > m_ref + kBias) {
              const float m_new = ceilf(top) - kBias;
              factor = m_ref == -INFINITY ? 1.f : exp2_approx(m_ref - m_new);     // O is zero or not begun: nothing to rescale
              m_ref = m_new;
            }
            moved = __any_sync(0xffffffffu, factor != 1.f);
          }
          if (!ok) break;
          l_sum = l_sum * factor + sum;
        }
        // O and both buffers for P are free when the P.V of the step before is done, here and there (a tile's last one was
        // waited for). Warps without rows wait as well: an arrival on p_full must not come before the last one was taken.
        if (k > 0 && !warp_wait(&ctl.pv_done, (g - 1) & 1, abort_flag, p.status, kWaitPv)) { ok = false; break; }
        if (warp_live) {
          if (moved && k > 0) {
            sm100::tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < kHalf; c += 32) {
              uint32_t o[32];
              sm100::tmem_ld_32x32(lanes + kColO + c, o);
              sm100::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st_32x32(lanes + kColO + c, o);
            }
            tmem_st_wait();
            sm100::tc_fence_before_sync();
          }
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(p_tile + row * 128 + ((c ^ (row & 7)) << 4)) =
                make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
          sm100::fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&ctl.p_full);
        // the same to the other CTA; in a tile's first step not before Q has come through the buffer there
        if (k == 0 && !warp_wait_peer(&ctl.x_first, (seg - 1) & 1, 0, abort_flag, p.status)) { ok = false; break; }
        if (lane == 0 && warp_live) bulk_copy_to(x_there, p_tile + warp * 32 * 128, 32 * 128, x_full_there);
        __syncwarp();
      }
      if (!ok) break;
      v_at += nb;
      if (nb > 0 && warp_live) send_word(sum_there, sum_full_there, __float_as_uint(l_sum));
      Walk nx = w;
      nx.next(p);
      if (nb > 0) {
        if (warp_live) {
          if (!warp_wait_peer(&ctl.sum_full[warp], sums & 1, 128, abort_flag, p.status)) { ok = false; break; }
          const float theirs = *reinterpret_cast<volatile float*>(&ctl.row_sum[row]);
          ++sums;
          l_sum = half == 0 ? l_sum + theirs : theirs + l_sum;
        }
        if (!warp_wait(&ctl.pv_done, (g - 1) & 1, abort_flag, p.status, kWaitPv)) { ok = false; break; }
        sm100::tc_fence_after_sync();
      }
      const bool whole = w.whole(), zero = l_sum == 0.f;
      const float inv = zero ? 0.f : 1.f / l_sum;              // NaN stays NaN
      const size_t slot = ((size_t)pair * 2 + (w.u0 == 0 ? 1 : 0)) * p.rows_cap + row;
      T* dst = static_cast<T*>(p.out) + (size_t)(w.t.row0 + row) * kDv + own;
      float4* part = p.part_o + ((slot - row) * (kDv / 4) + (size_t)(own / 4) * p.rows_cap + row);
#pragma unroll 1
      for (int c = 0; c < kHalf; c += 32) {
        if (c == kHalf / 2 && nb > 0) next_q(nx);              // by now it is there, and has its tensor cores busy meanwhile
        if (!ok) break;
        if (!warp_live) continue;
        uint32_t o[32];
        if (nb > 0) { sm100::tmem_ld_32x32(lanes + kColO + c, o); sm100::tmem_ld_wait(); }
        if (!live) continue;
        if (whole) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[k] = zero ? 0u : pack2<T>(__uint_as_float(o[8 * v + 2 * k]) * inv, __uint_as_float(o[8 * v + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + c + 8 * v) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else {                               // a cut tile has at least one step in each part
#pragma unroll
          for (int v = 0; v < 8; ++v)
            part[(size_t)(c / 4 + v) * p.rows_cap] = make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                                                                 __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
        }
      }
      if (!ok) break;
      if (live && whole && half == 0 && p.lse)
        p.lse[w.t.row0 + row] = zero ? -INFINITY : m_ref * 0.6931471805599453f + logf(l_sum);
      if (live && !whole && half == 0) p.part_ml[slot] = make_float2(m_ref, l_sum);
      sm100::tc_fence_before_sync();           // O was read: the next tile's first P.V comes after these threads' next p_full
      w = nx;
    }
    if (p.tail && ok) {                        // a warp per row; outside the division of work, so that padding does not move its cuts
      // (with wrong starts all rows are such; without sequences there is nothing before the tail)
      const long long end = (long long)p.T * p.H, begin = ctl.wrong || p.batch == 0 ? 0 : (long long)p.q_start[p.batch] * p.H;
      for (long long r = begin + blockIdx.x * 4 + warp; r < end; r += gridDim.x * 4) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + r * kDv);
        dst[lane] = dst[lane + 32] = make_uint4(0, 0, 0, 0);
        if (lane == 0 && p.lse) p.lse[r] = -INFINITY;
      }
    }
  }

  if (ctl.abort_flag) __nanosleep(50000);      // what is on its way to the other CTA lands
  sm100::tc_fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    sm100::tc_fence_after_sync();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
  __syncwarp();
  if (warp > 4) cluster_wait();
  sm100::cluster_sync_all();                   // nobody writes to a CTA that has ended
}

// Joins the parts of the tile that pair blockIdx.x ends: part k has weights relative to its own reference m_k. A block has
// eight rows, a thread of it four columns of each of its chunks of 128: all four chunks, or one where the grid has them as z.
// The parts are added in the order of the pairs. What costs is latency: eight loads are under way before the references
// and sums are waited for, kParts parts of 8 / kParts chunks.
constexpr int kMergeRows = 8, kMergeCols = 128, kMergeChunks = kDv / kMergeCols;
template <typename T, int kParts>
__device__ __forceinline__ void merge_parts(const Params& p, const Meta& m, float2 (&s_ml)[cab::kNumSMs / 2][kMergeRows]) {
  constexpr int kChunks = 8 / kParts;
  const int pair = blockIdx.x, sub = threadIdx.x % kMergeRows, row0 = blockIdx.y * kMergeRows, row = row0 + sub;
  const int parts = pair - m.first + 1, group = threadIdx.x / kMergeRows;
  const bool live = row < m.rows;
  auto slot_of = [&](int k) { return (size_t)(m.first + k) * 2 + (k == 0 ? 1 : 0); };
  float2 mine = make_float2(0.f, 0.f);         // at most one a thread in the first round, more parts follow below
  const int e0 = threadIdx.x / kMergeRows;
  if (e0 < parts && live) mine = p.part_ml[slot_of(e0) * p.rows_cap + row];
  float4 o[kChunks][kParts];
  auto load = [&](int c0, int k0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < kParts; ++e)
        if (live && k0 + e < parts && c0 + c < kMergeChunks)
          o[c][e] = __ldcs(p.part_o + (slot_of(k0 + e) * (kDv / 4) + (c0 + c) * (kMergeCols / 4) + group) * p.rows_cap + row);
  };
  load(blockIdx.z, 0);
  if (e0 < parts && live) s_ml[e0][sub] = mine;
  for (int k = e0 + kMergeCols / 4; k < parts; k += kMergeCols / 4)
    if (live) s_ml[k][sub] = p.part_ml[slot_of(k) * p.rows_cap + row];
  __syncthreads();
  if (!live) return;
  float top = -INFINITY;
  for (int k = 0; k < parts; ++k)
    if (s_ml[k][sub].y != 0.f) top = fmaxf(top, s_ml[k][sub].x);
  for (int c0 = blockIdx.z; c0 < kMergeChunks; c0 += gridDim.z * kChunks) {
    float4 acc[kChunks] = {};
    float l = 0.f;
    for (int k0 = 0; k0 < parts; k0 += kParts) {
      if (c0 != (int)blockIdx.z || k0 > 0) load(c0, k0);
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        if (k0 + e >= parts) break;
        const float2 ml = s_ml[k0 + e][sub];
        const float f = ml.y != 0.f ? exp2_approx(ml.x - top) : 0.f;
        if (f != 0.f) {                        // also true for NaN
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            acc[c].x += f * o[c][e].x; acc[c].y += f * o[c][e].y; acc[c].z += f * o[c][e].z; acc[c].w += f * o[c][e].w;
          }
          l += f * ml.y;
        }
      }
    }
    const bool zero = l == 0.f;
    const float inv = zero ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c0 + c >= kMergeChunks) break;
      uint2 r;
      r.x = zero ? 0u : pack2<T>(acc[c].x * inv, acc[c].y * inv);
      r.y = zero ? 0u : pack2<T>(acc[c].z * inv, acc[c].w * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (size_t)(m.row0 + row) * kDv + (c0 + c) * kMergeCols + group * 4) = r;
    }
    if (c0 == 0 && group == 0 && p.lse) p.lse[m.row0 + row] = zero ? -INFINITY : top * 0.6931471805599453f + logf(l);
  }
}
template <typename T>
__global__ void __launch_bounds__(kMergeRows * kMergeCols / 4, 4) mla_paged_merge_kernel(const Params p) {
  __shared__ float2 s_ml[cab::kNumSMs / 2][kMergeRows];
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  const Meta m = p.meta[blockIdx.x];
  if ((int)blockIdx.y * kMergeRows >= m.rows) return;
  const int parts = blockIdx.x - m.first + 1;
  if (gridDim.z > 1 || parts > 4) merge_parts<T, 8>(p, m, s_ml);
  else if (parts > 2) merge_parts<T, 4>(p, m, s_ml);
  else merge_parts<T, 2>(p, m, s_ml);
}

constexpr int kPairs = cab::kNumSMs / 2;       // the workspace is sized for this many, a smaller device runs fewer

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
int rows_cap_of(int T, int H) { return (int)((long long)T * H < kRows ? (long long)T * H : kRows); }

template <typename T>
int launch(Params& p, const Maps& maps, int sms, cudaStream_t stream) {
  if (!cab::ensure_dynamic_smem<&mla_paged_attention_kernel<T>>(kSmemBytes)) return CAB_ERR_LAUNCH;
  // Either kernel is set up while the one before it ends, and waits for that end itself before it reads or writes
  // anything (cudaGridDependencySynchronize): some 2 us less for a decode step.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * p.pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, mla_paged_attention_kernel<T>, static_cast<const Params>(p), maps) != cudaSuccess)
    return CAB_ERR_LAUNCH;
  if (p.pairs > 1) {
    // A chunk a block where there are so few rows that all their blocks run at once.
    const long long blocks = ((long long)p.T * p.H + kMergeRows - 1) / kMergeRows;
    cfg.gridDim = dim3(p.pairs, (p.rows_cap + kMergeRows - 1) / kMergeRows, blocks <= sms ? kMergeChunks : 1);
    cfg.blockDim = dim3(kMergeRows * kMergeCols / 4);
    cfg.dynamicSmemBytes = 0;
    if (cudaLaunchKernelEx(&cfg, mla_paged_merge_kernel<T>, static_cast<const Params>(p)) != cudaSuccess) return CAB_ERR_LAUNCH;
  }
  return cab::launch_status();
}

}  // namespace

extern "C" size_t mla_paged_attention_workspace_bytes(int T, int H) {
  if (T <= 0 || H <= 0) return 0;
  const size_t rows = (size_t)kPairs * 2 * rows_cap_of(T, H);
  return align256(rows * kDv * 4) + align256(rows * sizeof(float2)) + align256(kPairs * sizeof(Meta));
}

extern "C" int mla_paged_attention_launcher(void* out, float* lse, const void* q, const cab_mla_paged_batch* batch, int T,
                                            int H, float softmax_scale, int causal, int window, void* workspace,
                                            size_t workspace_bytes, int* status, int config, cudaStream_t stream) {
  if (T < 0 || H <= 0 || !batch || batch->batch < 0) return CAB_ERR_BAD_ARGUMENT;
  const bool tail = (config & 256) != 0;
  if (T == 0 || (batch->batch == 0 && !tail)) {
    if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
    return CAB_OK;
  }
  if (!out || !q || !workspace || !batch->rows || !batch->q_start ||
      (batch->batch > 0 && (!batch->page_table || !batch->kv_len)))
    return CAB_ERR_BAD_ARGUMENT;
  if (batch->num_pages <= 0 || batch->page_size <= 0 || batch->max_pages <= 0 || window < 0 || !(softmax_scale > 0.f) ||
      !(softmax_scale * kLog2e < 3.4e38f) || (batch->dtype != CAB_BF16 && batch->dtype != CAB_F16))
    return CAB_ERR_BAD_ARGUMENT;
  if (batch->page_stride % 8 || batch->token_stride % 8 || batch->token_stride < kD || batch->page_stride < kD)
    return CAB_ERR_BAD_ARGUMENT;
  if ((long long)T * H > 0x7fffffffLL || batch->batch > kMaxBatch) return CAB_ERR_TOO_LARGE;
  if ((long long)batch->max_pages * batch->page_size > 0x7fffff00LL) return CAB_ERR_TOO_LARGE;
  if (!cab::aligned_to(out, 16) || !cab::aligned_to(q, 16) || !cab::aligned_to(batch->rows, 16) ||
      !cab::aligned_to(workspace, 16))
    return CAB_ERR_MISALIGNED;
  if (workspace_bytes < mla_paged_attention_workspace_bytes(T, H)) return CAB_ERR_BAD_ARGUMENT;

  Params p;
  p.q = q; p.out = out; p.lse = lse;
  p.page_table = batch->page_table; p.q_start = batch->q_start; p.kv_len = batch->kv_len;
  p.T = T; p.H = H; p.batch = batch->batch; p.tail = tail;
  p.max_pages = batch->max_pages; p.num_pages = batch->num_pages; p.page_size = batch->page_size;
  // Rows that are sure to lie in one page, 64 at most. From eight on (the rows after which swizzling repeats) a box takes
  // all tiles of a part, and the tiles of eight rows lie after one another; below it is a box per tile.
  int box = 1;
  while (box < kKeys && batch->page_size % (2 * box) == 0) box *= 2;
  p.box = box;
  p.box_log2 = 0;
  while ((1 << p.box_log2) < box) ++p.box_log2;
  p.step_pages = kStep / batch->page_size; p.step_rows = kStep % batch->page_size;
  p.tile_bytes = box >= 8 ? 1024 : kTile;
  p.causal = causal != 0;
  p.window = window < (long long)batch->max_pages * batch->page_size ? window : 0;   // wider than any history: none
  p.rows_cap = rows_cap_of(T, H);
  p.scale_log2 = softmax_scale * kLog2e;
  const int sms = cab::sm_count();
  if (sms < 2) return CAB_ERR_LAUNCH;
  p.pairs = sms / 2 < kPairs ? sms / 2 : kPairs;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const size_t rows = (size_t)kPairs * 2 * p.rows_cap;
  p.part_o = reinterpret_cast<float4*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + align256(rows * kDv * 4));
  p.meta = reinterpret_cast<Meta*>(ws + align256(rows * kDv * 4) + align256(rows * sizeof(float2)));
  p.status = status;

  Maps maps;
  sm100::EncodeTiledFn encode = sm100::encode_tiled_fn();
  if (!encode) return CAB_ERR_LAUNCH;
  const CUtensorMapDataType type =
      batch->dtype == CAB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const bool eights = box >= 8;
  const cuuint64_t dims[5] = {64, (cuuint64_t)(eights ? 8 : batch->page_size), kD / 64, (cuuint64_t)(eights ? batch->page_size / 8 : 1),
                              (cuuint64_t)batch->num_pages};
  const cuuint64_t strides[4] = {(cuuint64_t)batch->token_stride * 2, 128, (cuuint64_t)batch->token_stride * 16,
                                 (cuuint64_t)batch->page_stride * 2};
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  auto make = [&](CUtensorMap* map, int tiles) {
    const cuuint32_t boxes[5] = {64, (cuuint32_t)(eights ? 8 : box), (cuuint32_t)tiles, (cuuint32_t)(eights ? box / 8 : 1), 1};
    return encode(map, type, 5, batch->rows, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (!make(&maps.one, 1) || !make(&maps.two, 2) || !make(&maps.four, 4)) return CAB_ERR_BAD_ARGUMENT;
  if (!sm100::make_tmap_2d_sw128(&maps.q, q, type, 2, (uint64_t)T * H, kD, kRows, 64) ||
      !sm100::make_tmap_2d_sw128(&maps.q16, q, type, 2, (uint64_t)T * H, kD, kQBox, 64))
    return CAB_ERR_BAD_ARGUMENT;
  if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
  return batch->dtype == CAB_F16 ? launch<__half>(p, maps, sms, stream) : launch<__nv_bfloat16>(p, maps, sms, stream);
}
