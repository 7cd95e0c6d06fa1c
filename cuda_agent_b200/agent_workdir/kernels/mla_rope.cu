// Rotary positions on a part of a head, and the same fused with the write of a batch's new rows into the paged
// latent cache.
//   (x0, x1) -> mscale * (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = position * freq[i]
// Memory bound: each column is read and written once. The angles depend on the token alone, so a CTA makes the
// sines and cosines of its tokens once, in shared memory, and uses them for all the heads it handles. The angle
// is formed and reduced to a fraction of a turn in 64 bits (at position 10^6 a 32-bit product is off by 0.03
// radian); sine and cosine of the fraction are 32-bit, as is the rotation; one rounding at the end.
// Columns move in 16-byte pieces where pointers, strides and R allow it, else pair by pair. A thread keeps one place
// in the row and steps through the rows of its CTA, so nothing is divided in the loop; its first rows are asked
// for before the sines and cosines are made.
// Measured: 64 of 576 bf16 columns of 4096 tokens x 128 heads, in halves, 24.9 us (5.4 TB/s of the 134 MB read and
// written; a library copy of the same strided view takes 24.7 us); 64 of 128 fp32 columns of 2047 tokens x 16 heads, inverse,
// 3.9 us; the append of 4096 tokens with 128 heads 31.8 us (144 MB, 4.5 TB/s: neither DRAM, 42 %, nor issue slots, 51 %, are
// full; its CTAs wait for starts and table entries before they write), of 32 tokens 6.0 us. (Per call, calls one behind the other.)
#include <cuda_fp16.h>

#include <type_traits>

#include "cab_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxR = 2048;
constexpr int kAngles = 1024;                  // sine / cosine pairs of a CTA

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values as one word: a conversion instruction rounds both.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 turn_of(int position, double freq, float mscale, bool inverse) {
  const double t = (double)position * (freq * 0.15915494309189533577);   // turns
  float s, c;
  sincospif((float)(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c * mscale, (inverse ? -s : s) * mscale);
}
__device__ __forceinline__ void rotate(float& a, float& b, float2 cs) {
  const float x = a * cs.x - b * cs.y, y = b * cs.x + a * cs.y;
  a = x;
  b = y;
}

// N elements that are one memory access.
template <typename T, int N>
struct __align__(sizeof(T) * N) Vec { T v[N]; };

// One unit of a head: with `interleaved` N consecutive columns (N / 2 pairs), else N columns of either half.
template <typename T, int N, bool kInterleaved>
struct Unit {
  static constexpr int kVecs = kInterleaved ? 1 : 2, kPairs = kInterleaved ? N / 2 : N;
  struct alignas(kPairs % 2 ? 8 : 16) Angles { float2 v[kPairs]; };
  Vec<T, N> d[kVecs];
  // `cs`: those of the token's first pair
  static __device__ __forceinline__ Angles angles(const float2* cs, int unit) {
    return *reinterpret_cast<const Angles*>(cs + unit * kPairs);
  }
  __device__ __forceinline__ void load(const T* x, int unit, int half) {
    d[0] = *reinterpret_cast<const Vec<T, N>*>(x + unit * N);
    if constexpr (!kInterleaved) d[1] = *reinterpret_cast<const Vec<T, N>*>(x + half + unit * N);
  }
  __device__ __forceinline__ void turn(const Angles& cs) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&d[0]);
      if constexpr (kInterleaved) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float2 x = unpack2<T>(w[i]);
          rotate(x.x, x.y, cs.v[i]);
          w[i] = pack2<T>(x.x, x.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float2 x = unpack2<T>(w[i]), y = unpack2<T>(w[N / 2 + i]);
          rotate(x.x, y.x, cs.v[2 * i]);
          rotate(x.y, y.y, cs.v[2 * i + 1]);
          w[i] = pack2<T>(x.x, x.y);
          w[N / 2 + i] = pack2<T>(y.x, y.y);
        }
      }
    } else if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float a = to_f(d[0].v[2 * i]), b = to_f(d[0].v[2 * i + 1]);
        rotate(a, b, cs.v[i]);
        d[0].v[2 * i] = from_f<T>(a);
        d[0].v[2 * i + 1] = from_f<T>(b);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float a = to_f(d[0].v[i]), b = to_f(d[kVecs - 1].v[i]);
        rotate(a, b, cs.v[i]);
        d[0].v[i] = from_f<T>(a);
        d[kVecs - 1].v[i] = from_f<T>(b);
      }
    }
  }
  __device__ __forceinline__ void store(T* x, int unit, int half) const {
    *reinterpret_cast<Vec<T, N>*>(x + unit * N) = d[0];
    if constexpr (!kInterleaved) *reinterpret_cast<Vec<T, N>*>(x + half + unit * N) = d[1];
  }
};

struct RopeParams {
  void* out;
  const void* x;
  const int* positions;
  const double* freq;
  int T, H, R, tokens;                         // tokens per CTA
  int heads;                                   // heads per CTA
  long long xt, xh, ot, oh;
  float mscale;
  int inverse;
};

// The rows (token, head) of a CTA, tokens x heads, of `units` units each: a thread takes the same unit of every
// (kThreads / units)-th row, four rows at a time.
template <typename T, int N, bool kInterleaved>
struct RowWalk {
  static constexpr int kBatch = kInterleaved ? 4 : 2;            // 64 bytes of a wide walk in flight per thread
  const T* x;
  T* out;
  int half, unit, tok, head, heads, left, step_tok, step_head;   // left: rows of this thread still to come
  long long xo, oo, x_step, o_step, x_wrap, o_wrap;
  Unit<T, N, kInterleaved> u[kBatch];
  long long at[kBatch];
  int cs_at[kBatch];

  __device__ __forceinline__ RowWalk(T* out_, const T* x_, int tokens, int heads_, int R, long long xt, long long xh,
                                     long long ot, long long oh)
      : x(x_), out(out_), half(R / 2), heads(heads_) {
    const int units = (kInterleaved ? R : half) / N;
    // (rows of more units than threads: the kernel comes again for the other units)
    const int step = units < kThreads ? kThreads / units : 1;
    unit = units < kThreads ? threadIdx.x % units : threadIdx.x;
    const int first = units < kThreads ? threadIdx.x / units : 0, rows = tokens * heads;
    left = first < step && first < rows ? (rows - first + step - 1) / step : 0;
    if (unit >= units) left = 0;
    tok = first / heads;
    head = first % heads;
    step_tok = step / heads;
    step_head = step % heads;
    xo = tok * xt + head * xh;
    oo = tok * ot + head * oh;
    x_step = step_tok * xt + step_head * xh;
    o_step = step_tok * ot + step_head * oh;
    x_wrap = xt - heads * xh;
    o_wrap = ot - heads * oh;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k < left) {
        u[k].load(x + xo, unit, half);
        at[k] = oo;
        cs_at[k] = tok * half;
      }
      xo += x_step;
      oo += o_step;
      tok += step_tok;
      head += step_head;
      if (head >= heads) {
        head -= heads;
        ++tok;
        xo += x_wrap;
        oo += o_wrap;
      }
    }
  }
  __device__ __forceinline__ void store(const float2* cs) {
    // the rows of a batch are mostly one token's, which turns them alike
    auto angles = Unit<T, N, kInterleaved>::angles(cs + cs_at[0], unit);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (k < left) {
        if (k > 0 && cs_at[k] != cs_at[k - 1]) angles = Unit<T, N, kInterleaved>::angles(cs + cs_at[k], unit);
        u[k].turn(angles);
        u[k].store(out + at[k], unit, half);
      }
    left -= kBatch;
  }
  __device__ __forceinline__ void rest(const float2* cs) {       // after the first load()
    while (left > 0) {
      store(cs);
      if (left > 0) load();
    }
  }
};

template <typename T, int N, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 4) mla_rope_kernel(const RopeParams p) {
  __shared__ __align__(16) float2 cs[kAngles];
  cab::after_predecessor();
  const int t0 = blockIdx.x * p.tokens, tokens = min(p.tokens, p.T - t0), half = p.R / 2;
  const int h0 = blockIdx.y * p.heads, h1 = min(p.H, h0 + p.heads);
  T* out = static_cast<T*>(p.out) + t0 * p.ot + h0 * p.oh;
  const T* x = static_cast<const T*>(p.x) + t0 * p.xt + h0 * p.xh;
  RowWalk<T, N, kInterleaved> w(out, x, tokens, h1 - h0, p.R, p.xt, p.xh, p.ot, p.oh);
  w.load();
  for (int e = threadIdx.x; e < tokens * half; e += kThreads)
    cs[e] = turn_of(p.positions[t0 + e / half], p.freq[e % half], p.mscale, p.inverse != 0);
  __syncthreads();
  w.rest(cs);
  // rows of more units than threads have: the others
  for (int unit = threadIdx.x + kThreads; unit < (kInterleaved ? p.R : half) / N; unit += kThreads) {
    RowWalk<T, N, kInterleaved> more(out, x, tokens, h1 - h0, p.R, p.xt, p.xh, p.ot, p.oh);
    more.unit = unit;
    more.left = tokens * (h1 - h0);
    more.load();
    more.rest(cs);
  }
}

constexpr int kLatent = 512, kRot = 64;

struct AppendParams {
  RopeParams r;                                // q: R = 64
  const void *c_kv, *k_pe;
  long long ct, kt;                            // token strides
  void* rows;
  long long page_stride, token_stride;
  int num_pages, page_size, batch, max_pages;
  const int *page_table, *q_start, *kv_len;
  int* status;
};

// kVec: every row and stride allows 16-byte accesses. Head group 0 of a token also writes the token's cache row.
template <typename T, bool kInterleaved, bool kVec>
__global__ void __launch_bounds__(kThreads, 4) mla_rope_append_kernel(const AppendParams p) {
  constexpr int N = kVec ? 8 : (kInterleaved ? 2 : 1);
  constexpr int half = kRot / 2;
  __shared__ __align__(16) float2 cs[kAngles];
  __shared__ int s_pos[kAngles / half];
  __shared__ long long s_row[kAngles / half];  // where the cache row begins, -1: nowhere
  cab::after_predecessor();
  const int t0 = blockIdx.x * p.r.tokens;
  const int end = min(max(p.q_start[p.batch], 0), p.r.T);     // tokens behind the last sequence stay as they are
  const int tokens = min(p.r.tokens, end - t0);
  const bool first = blockIdx.x == 0 && blockIdx.y == 0;
  if (tokens <= 0 && !first) return;           // the first one stays, to say whether the starts are sound
  // what does not depend on the tables is asked for before they are read
  const int h0 = blockIdx.y * p.r.heads, h1 = min(p.r.H, h0 + p.r.heads);
  RowWalk<T, N, kInterleaved> w(static_cast<T*>(p.r.out) + t0 * p.r.ot + h0 * p.r.oh,
                                static_cast<const T*>(p.r.x) + t0 * p.r.xt + h0 * p.r.xh, tokens, max(h1 - h0, 1), kRot,
                                p.r.xt, p.r.xh, p.r.ot, p.r.oh);
  if (h1 <= h0) w.left = 0;                    // no heads: only the cache is written
  w.load();
  constexpr int C = kVec ? 8 : 1;
  const T* c = static_cast<const T*>(p.c_kv) + t0 * p.ct;
  Vec<T, C> latent;
  const bool copies = blockIdx.y == 0;
  if (copies && threadIdx.x < tokens * (kLatent / C))
    latent = *reinterpret_cast<const Vec<T, C>*>(c + threadIdx.x / (kLatent / C) * p.ct + threadIdx.x % (kLatent / C) * C);
  // Wrong starts would put tokens on rows that are there already. Every CTA looks at all of them, so all agree to write nothing
  // (no difference up to 4096 sequences, their loads hide behind those of the rows; 16384 of one token with 128 heads 129 -> 169 us).
  bool wrong = false, lost = false;
#pragma unroll 4
  for (int b = kThreads - 1 - threadIdx.x; b < p.batch; b += kThreads)             // the last warps first: the first one has the search below
    wrong |= cab::wrong_start(p.q_start, b, p.batch, p.r.T);
  if (threadIdx.x < tokens) {
    const int t = t0 + threadIdx.x;
    int lo = 0, hi = p.batch;                  // last b with q_start[b] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const int pos = p.kv_len[lo] - p.q_start[lo + 1] + t;
    const int at = pos / p.page_size;
    const int page = pos >= 0 && at < p.max_pages ? p.page_table[(long long)lo * p.max_pages + at] : -1;
    const bool ok = (unsigned)page < (unsigned)p.num_pages;
    s_pos[threadIdx.x] = pos;
    s_row[threadIdx.x] = ok ? page * p.page_stride + (pos - at * p.page_size) * p.token_stride : -1;
    lost = !ok && blockIdx.y == 0;
  }
  if (__syncthreads_or(wrong)) {
    if (first && threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, (int)CAB_PAGED_BAD_INDEX);
    return;
  }
  if (lost && p.status) atomicCAS(p.status, 0, (int)CAB_PAGED_BAD_PAGE);
  for (int e = threadIdx.x; e < tokens * half; e += kThreads)
    cs[e] = turn_of(s_pos[e / half], p.r.freq[e % half], p.r.mscale, false);
  if (copies) {                                // the latent part of the rows: a copy
    T* rows = static_cast<T*>(p.rows);
    for (int e = threadIdx.x; e < tokens * (kLatent / C); e += kThreads) {
      const int t = e / (kLatent / C), col = e % (kLatent / C) * C;
      if (e != threadIdx.x) latent = *reinterpret_cast<const Vec<T, C>*>(c + t * p.ct + col);
      if (s_row[t] >= 0) *reinterpret_cast<Vec<T, C>*>(rows + s_row[t] + col) = latent;
    }
  }
  __syncthreads();
  if (copies) {
    constexpr int units = (kInterleaved ? kRot : half) / N;
    const T* k = static_cast<const T*>(p.k_pe) + t0 * p.kt;
    for (int e = threadIdx.x; e < tokens * units; e += kThreads) {
      const int t = e / units, unit = e % units;
      if (s_row[t] < 0) continue;
      Unit<T, N, kInterleaved> u;
      u.load(k + t * p.kt, unit, half);
      u.turn(Unit<T, N, kInterleaved>::angles(cs + t * half, unit));
      u.store(static_cast<T*>(p.rows) + s_row[t] + kLatent, unit, half);
    }
  }
  w.rest(cs);
}

// Tokens and heads per CTA: about `each` units a thread, fewer where the call is too small to fill the device. An append takes
// eight, so that its look into the tables is waited for less often (the large call above took 32.9 us, with four 36.9, with
// sixteen 33.5). The rotation alone takes four: on rows that another kernel or call just touched 26.6 us, with eight
// 27.4, with sixteen 28.5 (on rows that are nowhere near, 34.4, 33.6 and 31.4). These before launch_behind, 1.7 us each.
void split(RopeParams& p, int units_per_head, int each, dim3& grid) {
  const int half = p.R / 2;
  const long long per_token = (long long)(p.H > 0 ? p.H : 1) * units_per_head;
  long long tokens = each * kThreads / per_token;
  const long long most = kAngles / half < 1 ? 1 : kAngles / half;
  if (tokens > most) tokens = most;
  const long long fill = ((long long)p.T + 4 * cab::kNumSMs - 1) / (4 * cab::kNumSMs);
  if (tokens > fill) tokens = fill;
  if (tokens < 1) tokens = 1;
  p.tokens = (int)tokens;
  // a token alone is split over its heads when it is large, or when there are few tokens
  long long heads = p.H > 0 ? p.H : 1;
  if (tokens == 1) {
    const long long groups_wanted = p.T < 2 * cab::kNumSMs ? (2 * cab::kNumSMs + p.T - 1) / p.T : 1;
    long long smallest = 256 / units_per_head;                        // a thread has something to do
    if (smallest < 1) smallest = 1;
    heads = (heads + groups_wanted - 1) / groups_wanted;
    if (heads < smallest) heads = smallest;
    long long largest = 8 * kThreads / units_per_head;
    if (largest < 1) largest = 1;
    if (heads > largest) heads = largest;
  }
  p.heads = (int)heads;
  grid = dim3((unsigned)((p.T + tokens - 1) / tokens), (unsigned)(((p.H > 0 ? p.H : 1) + heads - 1) / heads));
}

template <typename T, int N, bool kInterleaved>
int launch_rope(RopeParams& p, cudaStream_t stream) {
  dim3 grid;
  split(p, (kInterleaved ? p.R : p.R / 2) / N, 4, grid);
  if (grid.y > 65535) return CAB_ERR_TOO_LARGE;
  return cab::launch_behind(&mla_rope_kernel<T, N, kInterleaved>, grid, dim3(kThreads), 0, stream, p);
}

template <typename T>
int run_rope(RopeParams& p, bool interleaved, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = cab::aligned_to(p.x, 16) && cab::aligned_to(p.out, 16) && p.xt % V == 0 && p.xh % V == 0 &&
                   p.ot % V == 0 && p.oh % V == 0 && (interleaved ? p.R : p.R / 2) % V == 0;
  if (interleaved) return vec ? launch_rope<T, V, true>(p, stream) : launch_rope<T, 2, true>(p, stream);
  return vec ? launch_rope<T, V, false>(p, stream) : launch_rope<T, 1, false>(p, stream);
}

template <typename T>
int run_append(AppendParams& p, bool interleaved, cudaStream_t stream) {
  auto vec16 = [](const void* q, long long a, long long b) { return cab::aligned_to(q, 16) && a % 8 == 0 && b % 8 == 0; };
  const bool vec = vec16(p.c_kv, p.ct, 0) && vec16(p.k_pe, p.kt, 0) &&
                   (p.r.H == 0 || (vec16(p.r.x, p.r.xt, p.r.xh) && vec16(p.r.out, p.r.ot, p.r.oh)));
  const int n = vec ? 8 : (interleaved ? 2 : 1);
  dim3 grid;
  split(p.r, (interleaved ? kRot : kRot / 2) / n, 8, grid);
  if (grid.y > 65535) return CAB_ERR_TOO_LARGE;
  if (interleaved)
    return vec ? cab::launch_behind(&mla_rope_append_kernel<T, true, true>, grid, dim3(kThreads), 0, stream, p)
               : cab::launch_behind(&mla_rope_append_kernel<T, true, false>, grid, dim3(kThreads), 0, stream, p);
  return vec ? cab::launch_behind(&mla_rope_append_kernel<T, false, true>, grid, dim3(kThreads), 0, stream, p)
             : cab::launch_behind(&mla_rope_append_kernel<T, false, false>, grid, dim3(kThreads), 0, stream, p);
}

}  // namespace

extern "C" int mla_rope_launcher(void* out, const void* x, const int* positions, const double* freq, int T, int H, int R,
                                 long long x_stride_t, long long x_stride_h, long long out_stride_t,
                                 long long out_stride_h, int dtype, int interleaved, int inverse, float mscale, int config,
                                 cudaStream_t stream) {
  (void)config;
  if (T < 0 || H < 0 || R <= 0 || R % 2) return CAB_ERR_BAD_ARGUMENT;
  if (T == 0 || H == 0) return CAB_OK;
  if (!out || !x || !positions || !freq) return CAB_ERR_BAD_ARGUMENT;
  if (R > kMaxR) return CAB_ERR_TOO_LARGE;
  const size_t element = dtype == CAB_F32 ? 4 : 2;
  // the pair by pair form takes the two columns of an interleaved pair as one access
  const size_t unit = interleaved ? 2 * element : element;
  if (!cab::aligned_to(x, unit) || !cab::aligned_to(out, unit) ||
      (interleaved && (x_stride_t % 2 || x_stride_h % 2 || out_stride_t % 2 || out_stride_h % 2)))
    return CAB_ERR_MISALIGNED;
  RopeParams p{out, x, positions, freq, T, H, R, 0, 0, x_stride_t, x_stride_h, out_stride_t, out_stride_h, mscale, inverse};
  switch (dtype) {
    case CAB_BF16: return run_rope<__nv_bfloat16>(p, interleaved != 0, stream);
    case CAB_F16: return run_rope<__half>(p, interleaved != 0, stream);
    case CAB_F32: return run_rope<float>(p, interleaved != 0, stream);
    default: return CAB_ERR_BAD_ARGUMENT;
  }
}

extern "C" int mla_rope_append_launcher(void* q_out, const void* q_pe, const void* c_kv, const void* k_pe,
                                        const cab_mla_paged_batch* batch, const double* freq, int T, int H,
                                        long long q_out_stride_t, long long q_out_stride_h, long long q_stride_t,
                                        long long q_stride_h, long long c_stride_t, long long k_stride_t, int interleaved,
                                        float mscale, int* status, int config, cudaStream_t stream) {
  (void)config;
  if (T < 0 || H < 0 || !batch || batch->batch < 0) return CAB_ERR_BAD_ARGUMENT;
  if (status && cudaMemsetAsync(status, 0, sizeof(int), stream) != cudaSuccess) return CAB_ERR_LAUNCH;
  if (T == 0 || batch->batch == 0) return CAB_OK;
  if (!c_kv || !k_pe || !freq || !batch->rows || !batch->page_table || !batch->q_start || !batch->kv_len ||
      (H > 0 && (!q_out || !q_pe)))
    return CAB_ERR_BAD_ARGUMENT;
  if (batch->num_pages <= 0 || batch->page_size <= 0 || batch->max_pages <= 0 || batch->page_stride % 8 ||
      batch->token_stride % 8 || batch->token_stride < kLatent + kRot)
    return CAB_ERR_BAD_ARGUMENT;
  if (!cab::aligned_to(batch->rows, 16)) return CAB_ERR_MISALIGNED;
  if (interleaved && (!cab::aligned_to(k_pe, 4) || k_stride_t % 2 ||
                      (H > 0 && (!cab::aligned_to(q_pe, 4) || !cab::aligned_to(q_out, 4) || q_stride_t % 2 ||
                                 q_stride_h % 2 || q_out_stride_t % 2 || q_out_stride_h % 2))))
    return CAB_ERR_MISALIGNED;
  AppendParams p;
  p.r = RopeParams{q_out, q_pe, nullptr, freq, T, H, kRot, 0, 0, q_stride_t, q_stride_h, q_out_stride_t, q_out_stride_h,
                   mscale, 0};
  p.c_kv = c_kv; p.k_pe = k_pe; p.ct = c_stride_t; p.kt = k_stride_t;
  p.rows = batch->rows; p.page_stride = batch->page_stride; p.token_stride = batch->token_stride;
  p.num_pages = batch->num_pages; p.page_size = batch->page_size; p.batch = batch->batch; p.max_pages = batch->max_pages;
  p.page_table = batch->page_table; p.q_start = batch->q_start; p.kv_len = batch->kv_len;
  p.status = status;
  switch (batch->dtype) {
    case CAB_BF16: return run_append<__nv_bfloat16>(p, interleaved != 0, stream);
    case CAB_F16: return run_append<__half>(p, interleaved != 0, stream);
    default: return CAB_ERR_BAD_ARGUMENT;
  }
}
