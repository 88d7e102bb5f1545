// Rotary positions computed from frequencies, and the append of a step's keys and values to a paged
// KV cache with that rotation applied on the way.
//
// Mathematics.  Pair i of a head at position p turns by a = p * inv_freq[i]; (x0, x1) becomes
// s (x0 cos a - x1 sin a, x1 cos a + x0 sin a) with the caller's scale s; pairs are (i, i + R/2)
// (half layout) or (2i, 2i + 1) (interleaved); the D - R values behind them are copied.  The backward
// pass is the transposed matrix: the same with -a.  The angle is formed and reduced to a fraction of a
// turn in 64 bits (at position 10^6 a 32-bit angle is off by 0.03 radian), its sine and cosine and the
// rotation are 32-bit, and each output is rounded once.
//
// What bounds it: memory traffic (every value read and written once).  So: 16-byte accesses; one launch for queries
// and keys (and values, where they go to the pages); a block for a token, which forms its R/2 angles once in LDS and
// uses them for every head, so the 64-bit arithmetic is paid per token and pair and not per head.  The first loads are
// on their way before the angles (and the token's place in the pages: three dependent loads) are known; with that,
// blocks of 2 to 4 tokens are slower (8192 tokens of 80 heads of 128 in bf16: 67 us with one token a block, 69 with 2
// or 4; 8340 tokens of 48 heads of 64 to pages of 16: 31, 35, 39 us).
// Measured: 66 us for 0.34 GB read and written (5.1 TB/s); 22 us for 0.11 GB, a quarter of each head turned (5.2 TB/s);
// 30 us for the 8340 tokens' 0.10 GB (3.4 TB/s: two loads a thread behind the place and the angles); 4 us for 16
// tokens, a launch.
#include "paged.h"

namespace pa {
namespace rot {

constexpr int kMaxPairs = 256;  // R / 2 of one token

__device__ __forceinline__ float2 angle(const double* inv_freq, float scale, long long p, int i, float sign) {
  float c, s;
  const double turns = (double)p * inv_freq[i] * 0.15915494309189533577;  // / 2 pi
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c * scale, sign * s * scale);
}

// Units of a head: `nr` that turn (V values and their V partners at + pairs in the half layout, V values of
// interleaved pairs), then the copied ones of V values.  A thread's units of the block's token, in order:
struct Walk {
  int threads, units, nr, heads, Ht;  // heads: taken at once
  int u, hh, hl;             // the next unit, its head
  bool more;
  __device__ __forceinline__ Walk(int V, bool inter, int D, int pairs, int Ht_, int threads_) {
    threads = threads_;
    nr = (inter ? 2 * pairs : pairs) / V;
    units = nr + (D - 2 * pairs) / V;
    heads = units < threads ? threads / units : 1;
    Ht = Ht_;
    hl = threadIdx.x / units;
    u = threadIdx.x % units;
    hh = hl;
    more = hl < heads && hl < Ht;
  }
  __device__ __forceinline__ void next() {
    hh += heads;
    if (hh < Ht) return;
    hh = hl;
    u += threads;  // only where a head has more units than the block threads
    more = u < units;
  }
  template <int V, bool INTER>
  __device__ __forceinline__ int off(int pairs) const {
    return INTER || u < nr ? u * V : 2 * pairs + (u - nr) * V;
  }
};

// One unit turned (or copied), with the bias on it.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void turn_unit(const Pack<T, V>& x, const Pack<T, V>& x2, T* __restrict__ y,
                                          const T* __restrict__ bias, const float2* __restrict__ cs, int half, bool turn,
                                          bool two) {
  float a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = to_f(x.v[e]);
  if (bias) {
    float t[V];
    load_f<T, V>(bias, t);
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] += t[e];
  }
  if constexpr (INTER) {
    if (turn) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 c = cs[e / 2];
        const float u = a[e], v = a[e + 1];
        a[e] = u * c.x - v * c.y;
        a[e + 1] = v * c.x + u * c.y;
      }
    }
    store_f<T, V>(y, a);
  } else {
    if (two) {
#pragma unroll
      for (int e = 0; e < V; ++e) b[e] = to_f(x2.v[e]);
      if (bias) {
        float t[V];
        load_f<T, V>(bias + half, t);
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] += t[e];
      }
      if (turn) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 c = cs[e];
          const float u = a[e], v = b[e];
          a[e] = u * c.x - v * c.y;
          b[e] = v * c.x + u * c.y;
        }
      }
      store_f<T, V>(y + half, b);
    }
    store_f<T, V>(y, a);
  }
}

// A block's units, G loads of a thread in flight; the first ones are on their way while `before` forms the angles.
template <typename T, int V, bool INTER, int G, typename Src, typename Before, typename Put>
__device__ __forceinline__ void stream(Walk w, int pairs, Src src, Before before, Put put) {
  Pack<T, V> a[G], b[G];
  Walk ahead = w;
  auto load = [&]() {
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (ahead.more) {
        const T* x = src(ahead.hh) + ahead.template off<V, INTER>(pairs);
        a[j] = *reinterpret_cast<const Pack<T, V>*>(x);
        if (!INTER && ahead.u < w.nr) b[j] = *reinterpret_cast<const Pack<T, V>*>(x + pairs);
        ahead.next();
      }
  };
  load();
  before();
  while (w.more) {
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (w.more) {
        put(w.hh, w.template off<V, INTER>(pairs), w.u < w.nr, a[j], b[j]);
        w.next();
      }
    load();
  }
}

struct RopeArgs {
  const void* x[2];
  void* y[2];
  long long xs[2][3];  // batch, token, head strides of the inputs; the outputs are contiguous
  int H[2];
  const void* pos;  // int32 / int64 [B, S] of the given strides, or null: the token's index
  long long ps[2];
  int pos64;
  int S, D, pairs, threads;
  long long tokens;
  float sign, scale;
  const double* inv_freq;
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs A) {
  __shared__ float2 cs[kMaxPairs];
  const long long tok = blockIdx.x;
  const int b = blockIdx.x / A.S, s = blockIdx.x - b * A.S;
  const T* const x0 = reinterpret_cast<const T*>(A.x[0]) + b * A.xs[0][0] + s * A.xs[0][1];
  const T* const x1 = reinterpret_cast<const T*>(A.x[1]) + b * A.xs[1][0] + s * A.xs[1][1];
  T* const y0 = reinterpret_cast<T*>(A.y[0]) + tok * A.H[0] * A.D;
  T* const y1 = reinterpret_cast<T*>(A.y[1]) + tok * A.H[1] * A.D;
  stream<T, V, INTER, 4>(
      Walk(V, INTER, A.D, A.pairs, A.H[0] + A.H[1], A.threads), A.pairs,
      [&](int hh) { return hh < A.H[0] ? x0 + hh * A.xs[0][2] : x1 + (hh - A.H[0]) * A.xs[1][2]; },
      [&]() {
        long long p = s;
        if (A.pos)
          p = A.pos64 ? reinterpret_cast<const int64_t*>(A.pos)[b * A.ps[0] + s * A.ps[1]]
                      : (long long)reinterpret_cast<const int32_t*>(A.pos)[b * A.ps[0] + s * A.ps[1]];
        for (int i = threadIdx.x; i < A.pairs; i += A.threads) cs[i] = angle(A.inv_freq, A.scale, p, i, A.sign);
        __syncthreads();
      },
      [&](int hh, int off, bool turn, const Pack<T, V>& a, const Pack<T, V>& b) {
        T* y = (hh < A.H[0] ? y0 + (long long)hh * A.D : y1 + (long long)(hh - A.H[0]) * A.D) + off;
        turn_unit<T, V, INTER>(a, b, y, (const T*)nullptr, &cs[INTER ? off / 2 : off], A.pairs, turn, turn);
      });
}

struct AppendArgs {
  const void* qkv;
  long long row;  // stride of a token's row
  const void* bias;
  void* q;  // [T, Hq, D]
  void* kc;
  void* vc;
  long long cs[3];  // block, head, slot strides of both caches
  const int* tables;
  long long tstride;
  int max_blocks, num_blocks, page;
  const int* lens;  // tokens cached before this call
  const int* cu;    // [B + 1] or null: one token each
  const void* off_dev;  // int32 / int64 or null
  int off64;
  long long off;  // position = off + place in the cache
  int T, B, Hq, Hkv, D, pairs, threads;
  float scale;
  const double* inv_freq;
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs A) {
  __shared__ float2 cs[kMaxPairs];
  const int t = blockIdx.x;
  const T* const x = reinterpret_cast<const T*>(A.qkv) + (long long)t * A.row;
  T* const q = reinterpret_cast<T*>(A.q) + (long long)t * A.Hq * A.D;
  bool in = false;     // the token belongs to a sequence
  long long dst = -1;  // where its keys go (element offset of head 0), -1: nowhere
  stream<T, V, INTER, 4>(
      Walk(V, INTER, A.D, A.pairs, A.Hq + 2 * A.Hkv, A.threads), A.pairs, [&](int hh) { return x + (long long)hh * A.D; },
      [&]() {
        // (each wave for itself: no barrier before the angles)
        const int b = A.cu ? __builtin_amdgcn_readfirstlane(seq_of_token(A.cu, A.B, t)) : (t < A.B ? t : A.B);
        in = b >= 0 && b < A.B;
        if (in) {
          long long p = (long long)A.lens[b] + (A.cu ? t - A.cu[b] : 0);
          const long long pg = p / A.page;
          if (p >= 0 && pg < A.max_blocks) {
            const int blk = A.tables[(long long)b * A.tstride + pg];
            if (blk >= 0 && blk < A.num_blocks) dst = blk * A.cs[0] + (p - pg * A.page) * A.cs[2];
          }
          p += !A.off_dev ? A.off
                          : (A.off64 ? *reinterpret_cast<const int64_t*>(A.off_dev)
                                     : (long long)*reinterpret_cast<const int32_t*>(A.off_dev));
          for (int i = threadIdx.x; i < A.pairs; i += A.threads) cs[i] = angle(A.inv_freq, A.scale, p, i, 1.f);
        }
        __syncthreads();
      },
      [&](int hh, int off, bool turn, const Pack<T, V>& a, const Pack<T, V>& b) {
        T* y;
        if (hh < A.Hq) {
          y = q + (long long)hh * A.D + off;
          if (!in) {  // behind the last sequence
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = 0.f;
            store_f<T, V>(y, z);
            if (!INTER && turn) store_f<T, V>(y + A.pairs, z);
            return;
          }
        } else {
          if (dst < 0) return;
          const bool isv = hh >= A.Hq + A.Hkv;
          const int h = hh - A.Hq - (isv ? A.Hkv : 0);
          y = reinterpret_cast<T*>(isv ? A.vc : A.kc) + dst + h * A.cs[1] + off;
        }
        const T* bias = A.bias ? reinterpret_cast<const T*>(A.bias) + (long long)hh * A.D + off : nullptr;
        turn_unit<T, V, INTER>(a, b, y, bias, &cs[INTER ? off / 2 : off], A.pairs, turn && hh < A.Hq + A.Hkv, turn);
      });
}

// Vector width: the widest of 16, 8, 4 ... bytes that divides the pairs, the copied part and, by the
// caller's word, every stride and address (`align` elements).
inline int width(int esz, int D, int pairs, bool inter, int align) {
  int v = 16 / esz;
  while (v > (inter ? 2 : 1) && ((inter ? 2 * pairs : pairs) % v || D % v || (D - 2 * pairs) % v || align % v)) v >>= 1;
  return v;
}

}  // namespace rot
}  // namespace pa

using namespace pa::rot;

#define PA_ROT_LAUNCH(T, KERNEL, ...)                                                            \
  if (inter) {                                                                                   \
    if (v == 8) { if constexpr (sizeof(T) == 2) KERNEL<T, 8, true> __VA_ARGS__; }                \
    else if (v == 4) KERNEL<T, 4, true> __VA_ARGS__;                                             \
    else KERNEL<T, 2, true> __VA_ARGS__;                                                         \
  } else {                                                                                       \
    if (v == 8) { if constexpr (sizeof(T) == 2) KERNEL<T, 8, false> __VA_ARGS__; }               \
    else if (v == 4) KERNEL<T, 4, false> __VA_ARGS__;                                            \
    else if (v == 2) KERNEL<T, 2, false> __VA_ARGS__;                                            \
    else KERNEL<T, 1, false> __VA_ARGS__;                                                        \
  }

// Threads of a token's block: two units a thread, up to 4 waves (65536 tokens of 4 + 4 heads of 64, 32 units: 31 us with
// one wave, 44 with two, 69 with four; 32768 of 8 + 2 heads of 128, 80 units: 27, 30, 43; from 320 units on four waves
// are as fast as one, and for few tokens faster: 16 of 48 heads of 128, 384 units: 6.2, 4.8, 4.2).  An argument of the
// kernel: the block's size as the hardware tells it is a load more before the first data (80 heads of 128: 64 beside 61 us).
inline int block_threads(int D, int pairs, bool inter, int heads, int v) {
  const long long units = (long long)heads * ((inter ? 2 * pairs : pairs) / v + (D - 2 * pairs) / v);
  return units <= 128 ? 64 : (units <= 256 ? 128 : 256);
}

// q / k: [B, S, H, D] views with unit inner stride and the given (batch, token, head) strides; yq / yk
// contiguous.  `align`: elements that divide every stride and address.  sign -1: the backward pass.
PA_API int pa_rope_freq(const void* q, const void* k, void* yq, void* yk, const long long* qs, const long long* ks,
                        int B, int S, int Hq, int Hk, int D, int pairs, int inter, const double* inv_freq, float scale,
                        const void* pos, long long pos_b, long long pos_s, int pos64, float sign, int align, int dt,
                        hipStream_t st) {
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || pairs < 0 || 2 * pairs > D || pairs > kMaxPairs || align < 1)
    return (int)hipErrorInvalidValue;
  RopeArgs A;
  A.x[0] = q; A.x[1] = k; A.y[0] = yq; A.y[1] = yk;
  for (int i = 0; i < 3; ++i) { A.xs[0][i] = qs[i]; A.xs[1][i] = ks ? ks[i] : 0; }
  A.H[0] = Hq; A.H[1] = k ? Hk : 0;
  A.pos = pos; A.ps[0] = pos_b; A.ps[1] = pos_s; A.pos64 = pos64;
  A.S = S; A.D = D; A.pairs = pairs; A.tokens = (long long)B * S; A.sign = sign;
  A.inv_freq = inv_freq; A.scale = scale;
  if (A.tokens == 0 || A.H[0] + A.H[1] == 0) return 0;
  const int v = width(dt == 0 ? 4 : 2, D, pairs, inter != 0, align);
  if (inter && (D % v || align % v)) return (int)hipErrorInvalidValue;  // pairs are loaded together
  if (A.tokens > 0x7fffffff) return (int)hipErrorInvalidValue;
  A.threads = block_threads(D, pairs, inter != 0, A.H[0] + A.H[1], v);
  PA_DISPATCH_DTYPE(dt, T, PA_ROT_LAUNCH(T, rope_kernel, <<<(int)A.tokens, A.threads, 0, st>>>(A)))
  return (int)hipGetLastError();
}

// qkv rows [T, (Hq + 2 Hkv) D] (+ bias) -> q [T, Hq, D] turned, keys (turned) and values into the pages.
// The angle's position: off or *off_dev, + place.
PA_API int pa_paged_append(const void* qkv, long long row, const void* bias, void* q, void* kc, void* vc,
                           const long long* cstr, const int* tables, long long tstride, int max_blocks, int num_blocks,
                           int page, const int* lens, const int* cu, const void* off_dev, int off64, long long off,
                           int T, int B, int Hq, int Hkv, int D, int pairs, int inter, const double* inv_freq,
                           float scale, int align, int dt, hipStream_t st) {
  if (T < 0 || B < 0 || Hq < 0 || Hkv <= 0 || D <= 0 || pairs < 0 || 2 * pairs > D || pairs > kMaxPairs || page <= 0 ||
      align < 1 || (pairs > 0 && !inv_freq))
    return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  AppendArgs A;
  A.qkv = qkv; A.row = row; A.bias = bias; A.q = q; A.kc = kc; A.vc = vc;
  for (int i = 0; i < 3; ++i) A.cs[i] = cstr[i];
  A.tables = tables; A.tstride = tstride; A.max_blocks = max_blocks; A.num_blocks = num_blocks; A.page = page;
  A.lens = lens; A.cu = cu; A.off_dev = off_dev; A.off64 = off64; A.off = off;
  A.T = T; A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.pairs = pairs;
  A.inv_freq = inv_freq; A.scale = scale;
  const int v = width(dt == 0 ? 4 : 2, D, pairs, inter != 0, align);
  if (inter && (D % v || align % v)) return (int)hipErrorInvalidValue;
  A.threads = block_threads(D, pairs, inter != 0, Hq + 2 * Hkv, v);
  PA_DISPATCH_DTYPE(dt, T_, PA_ROT_LAUNCH(T_, append_kernel, <<<T, A.threads, 0, st>>>(A)))
  return (int)hipGetLastError();
}
