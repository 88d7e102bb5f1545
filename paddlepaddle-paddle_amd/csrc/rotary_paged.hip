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
// What bounds it: memory traffic (every value read and written once).  So: 16-byte accesses; one launch
// for queries and keys (and values, where they go to the pages); a block takes 1 or 4 tokens, forms
// their R/2 angles once in LDS and uses them for every head, so the 64-bit arithmetic is paid per token
// and pair and not per head.
#include "common.h"

namespace pa {
namespace rot {

constexpr int kMaxPairs = 256;  // R / 2 of one token

// cos/sin of a position's pairs: from frequencies, or from tables[(b, p, i)] of the given length
struct Angles {
  const double* inv_freq;
  const float* cos_t;
  const float* sin_t;
  long long tab_b;  // table stride of a sequence
  int tab_len;      // positions per table
  float scale;
};

__device__ __forceinline__ float2 angle(const Angles& a, int b, long long p, int i, int pairs, float sign) {
  float c, s;
  if (a.cos_t != nullptr) {
    if (p < 0 || p >= a.tab_len) return make_float2(NAN, NAN);  // no such row: loud, and never read
    const long long o = (long long)b * a.tab_b + p * pairs + i;
    c = a.cos_t[o];
    s = a.sin_t[o];
  } else {
    const double turns = (double)p * a.inv_freq[i] * 0.15915494309189533577;  // / 2 pi
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    c *= a.scale;
    s *= a.scale;
  }
  return make_float2(c, sign * s);
}

// One vector unit of a head: V values (interleaved pairs, or values that are copied), or the V values at
// x and their V partners at x + half.  No contraction: a product is rounded before it is added, as in
// the composite of elementary operations.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void turn_unit(const T* __restrict__ x, T* __restrict__ y, const T* __restrict__ bias,
                                          const float2* __restrict__ cs, int half, bool turn, bool two) {
#pragma clang fp contract(off)
  float a[V], b[V];
  load_f<T, V>(x, a);
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
      load_f<T, V>(x + half, b);
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

// Units of a head: `nr` that turn (each V values and their partners in the half layout, V values
// interleaved), then the copied ones.  Offset of unit u within the head:
template <int V, bool INTER>
__device__ __forceinline__ int unit_off(int u, int nr, int pairs) {
  return INTER ? u * V : (u < nr ? u * V : 2 * pairs + (u - nr) * V);
}

struct RopeArgs {
  const void* x[2];
  void* y[2];
  long long xs[2][3];  // batch, token, head strides of the inputs; the outputs are contiguous
  int H[2];
  const void* pos;  // int32 / int64 [B, S] of the given strides, or null: the token's index
  long long ps[2];
  int pos64;
  int S, D, pairs;
  long long tokens;
  float sign;
  Angles ang;
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs A, int per_block) {
  __shared__ float2 cs[4][kMaxPairs];
  const long long t0 = (long long)blockIdx.x * per_block;
  const int nt = (int)min((long long)per_block, A.tokens - t0);
  for (int i = threadIdx.x; i < nt * A.pairs; i += 256) {
    const int t = i / A.pairs, j = i - t * A.pairs;
    const long long tok = t0 + t, b = tok / A.S, s = tok - b * A.S;
    long long p = s;
    if (A.pos)
      p = A.pos64 ? reinterpret_cast<const int64_t*>(A.pos)[b * A.ps[0] + s * A.ps[1]]
                  : (long long)reinterpret_cast<const int32_t*>(A.pos)[b * A.ps[0] + s * A.ps[1]];
    cs[t][j] = angle(A.ang, 0, p, j, A.pairs, A.sign);
  }
  __syncthreads();
  const int nr = INTER ? 2 * A.pairs / V : A.pairs / V;
  const int units = nr + (A.D - 2 * A.pairs) / V;
  const int Ht = A.H[0] + A.H[1];
  const int heads = 256 / units > 0 ? 256 / units : 1;  // heads that the block takes at once
  const int hl = threadIdx.x / units;
  for (int u = threadIdx.x % units; u < units; u += 256) {  // more than once only where a head has over 256 units
    const int off = unit_off<V, INTER>(u, nr, A.pairs);
    if (hl >= heads) break;
    for (int t = 0; t < nt; ++t) {
      const long long tok = t0 + t, b = tok / A.S, s = tok - b * A.S;
      for (int hh = hl; hh < Ht; hh += heads) {
        const int w = hh < A.H[0] ? 0 : 1, h = w ? hh - A.H[0] : hh;
        const T* x = reinterpret_cast<const T*>(w ? A.x[1] : A.x[0]) + b * (w ? A.xs[1][0] : A.xs[0][0]) +
                     s * (w ? A.xs[1][1] : A.xs[0][1]) + h * (w ? A.xs[1][2] : A.xs[0][2]) + off;
        T* y = reinterpret_cast<T*>(w ? A.y[1] : A.y[0]) + (tok * (w ? A.H[1] : A.H[0]) + h) * (long long)A.D + off;
        turn_unit<T, V, INTER>(x, y, (const T*)nullptr, &cs[t][INTER ? off / 2 : off], A.pairs, u < nr, u < nr);
      }
    }
  }
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
  const int* off_dev;
  long long off;  // position = off + place in the cache
  int T, B, Hq, Hkv, D, pairs;
  Angles ang;
};

// largest b with cu[b] <= t, or B where t lies behind the last sequence (-1 before the first)
__device__ __forceinline__ int seq_of_token(const int* cu, int B, int t) {
  if (t >= cu[B]) return B;
  int lo = -1, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs A, int per_block) {
  __shared__ float2 cs[4][kMaxPairs];
  __shared__ long long dst[4];  // where the token's keys go (element offset of head 0), -1: nowhere
  __shared__ long long where[4];
  __shared__ int seq[4];
  const int t0 = blockIdx.x * per_block, nt = min(per_block, A.T - t0);
  if (threadIdx.x < nt) {
    const int t = t0 + threadIdx.x;
    const int b = A.cu ? seq_of_token(A.cu, A.B, t) : (t < A.B ? t : A.B);
    long long d = -1, p = 0;
    int s = -1;
    if (b >= 0 && b < A.B) {
      s = b;
      p = (long long)A.lens[b] + (A.cu ? t - A.cu[b] : 0);
      const long long pg = p / A.page;
      if (p >= 0 && pg < A.max_blocks) {
        const int blk = A.tables[(long long)b * A.tstride + pg];
        if (blk >= 0 && blk < A.num_blocks) d = blk * A.cs[0] + (p - pg * A.page) * A.cs[2];
      }
      p += A.off_dev ? (long long)*A.off_dev : A.off;
    }
    dst[threadIdx.x] = d;
    where[threadIdx.x] = p;
    seq[threadIdx.x] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nt * A.pairs; i += 256) {
    const int t = i / A.pairs, j = i - t * A.pairs;
    if (seq[t] >= 0) cs[t][j] = angle(A.ang, seq[t], where[t], j, A.pairs, 1.f);
  }
  __syncthreads();
  const int nr = INTER ? 2 * A.pairs / V : A.pairs / V;
  const int units = nr + (A.D - 2 * A.pairs) / V;
  const int Ht = A.Hq + 2 * A.Hkv;
  const int heads = 256 / units > 0 ? 256 / units : 1;
  const int hl = threadIdx.x / units;
  for (int u = threadIdx.x % units; u < units; u += 256) {
    const int off = unit_off<V, INTER>(u, nr, A.pairs);
    if (hl >= heads) break;
    for (int t = 0; t < nt; ++t) {
      const long long tok = t0 + t;
      for (int hh = hl; hh < Ht; hh += heads) {
        const long long o = (long long)hh * A.D + off;
        const T* x = reinterpret_cast<const T*>(A.qkv) + tok * A.row + o;
        const T* bias = A.bias ? reinterpret_cast<const T*>(A.bias) + o : nullptr;
        T* y;
        if (hh < A.Hq) {
          y = reinterpret_cast<T*>(A.q) + (tok * A.Hq + hh) * (long long)A.D + off;
          if (seq[t] < 0) {  // behind the last sequence
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = 0.f;
            store_f<T, V>(y, z);
            if (!INTER && u < nr) store_f<T, V>(y + A.pairs, z);
            continue;
          }
        } else {
          if (dst[t] < 0) continue;
          const bool isv = hh >= A.Hq + A.Hkv;
          const int h = hh - A.Hq - (isv ? A.Hkv : 0);
          y = reinterpret_cast<T*>(isv ? A.vc : A.kc) + dst[t] + h * A.cs[1] + off;
        }
        turn_unit<T, V, INTER>(x, y, bias, &cs[t][INTER ? off / 2 : off], A.pairs, u < nr && hh < A.Hq + A.Hkv, u < nr);
      }
    }
  }
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

// Tokens per block: 4 once that still gives every CU two blocks (the angles of 4 tokens fill the
// block's 256 threads at R = 128), else 1, which spreads a decode step over the chip.
static int rot_tokens_per_block(long long tokens) { return tokens >= 2048 ? 4 : 1; }

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
  A.ang = Angles{inv_freq, nullptr, nullptr, 0, 0, scale};
  if (A.tokens == 0 || A.H[0] + A.H[1] == 0) return 0;
  const int v = width(dt == 0 ? 4 : 2, D, pairs, inter != 0, align);
  if (inter && (D % v || align % v)) return (int)hipErrorInvalidValue;  // pairs are loaded together
  const int pb = rot_tokens_per_block(A.tokens);
  const long long grid = (A.tokens + pb - 1) / pb;
  if (grid > 0x7fffffff) return (int)hipErrorInvalidValue;
  PA_DISPATCH_DTYPE(dt, T, PA_ROT_LAUNCH(T, rope_kernel, <<<(int)grid, 256, 0, st>>>(A, pb)))
  return (int)hipGetLastError();
}

// qkv rows [T, (Hq + 2 Hkv) D] (+ bias) -> q [T, Hq, D] turned, keys (turned) and values into the pages.
// Angles from inv_freq (position = off or *off_dev + place), or from cos / sin tables [B, tab_len, pairs].
PA_API int pa_paged_append(const void* qkv, long long row, const void* bias, void* q, void* kc, void* vc,
                           const long long* cstr, const int* tables, long long tstride, int max_blocks, int num_blocks,
                           int page, const int* lens, const int* cu, const int* off_dev, long long off, int T, int B,
                           int Hq, int Hkv, int D, int pairs, int inter, const double* inv_freq, float scale,
                           const float* cos_t, const float* sin_t, long long tab_b, int tab_len, int align, int dt,
                           hipStream_t st) {
  if (T < 0 || B < 0 || Hq < 0 || Hkv <= 0 || D <= 0 || pairs < 0 || 2 * pairs > D || pairs > kMaxPairs || page <= 0 ||
      align < 1 || (pairs > 0 && !inv_freq && !(cos_t && sin_t)))
    return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  AppendArgs A;
  A.qkv = qkv; A.row = row; A.bias = bias; A.q = q; A.kc = kc; A.vc = vc;
  for (int i = 0; i < 3; ++i) A.cs[i] = cstr[i];
  A.tables = tables; A.tstride = tstride; A.max_blocks = max_blocks; A.num_blocks = num_blocks; A.page = page;
  A.lens = lens; A.cu = cu; A.off_dev = off_dev; A.off = off;
  A.T = T; A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.pairs = pairs;
  A.ang = Angles{inv_freq, cos_t, sin_t, tab_b, tab_len, scale};
  const int v = width(dt == 0 ? 4 : 2, D, pairs, inter != 0, align);
  if (inter && (D % v || align % v)) return (int)hipErrorInvalidValue;
  const int pb = rot_tokens_per_block(T);
  PA_DISPATCH_DTYPE(dt, T_, PA_ROT_LAUNCH(T_, append_kernel, <<<(T + pb - 1) / pb, 256, 0, st>>>(A, pb)))
  return (int)hipGetLastError();
}
