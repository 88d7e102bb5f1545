// Sampling of one token per row from filtered logits with given random numbers.
//
// Mathematics.  w_i = exp((x_i - max x) / t).  The kept set is, of the tokens in the order of falling x
// (equal x: the lower index first), the first k; of those the ones before which less than p of their mass
// lies (at least one); of those the ones with w_i >= m.  The answer is the first token, in the order of the
// vocabulary, at which the kept mass passes u times its total.  Tokens of -inf or NaN are never kept.
//
// No sort, and one read of the logits by the whole chip.  Two kernels:
//  * chunk_kernel, a block for 8192 tokens of a row: their maximum, and a histogram of counts and masses over
//    bins of 1/8 in log2 w (a grid of absolute log2 w, so that the chunks' bins line up);
//  * row_kernel, a block for a row: the chunks' histograms joined, the bins in which the k-th token, the share
//    p and the border of min-p lie, the few tokens of those bins gathered and ranked, the chunk in which the
//    kept mass passes its goal, and a scan of that chunk.
// A bin of more than 1024 tokens at a border (ties, flat rows) takes radix selection over the whole row instead.
//
// Weights are 64-bit floats: a 32-bit sum over 10^5 tokens moves the borders of the cumulative distribution
// by more than a token's share.  Masses that are added by atomics are 64-bit integers (w scaled by 2^S with S
// so large that the sum just fits), so the answer does not depend on their order.  Tokens under 2^-47 of the
// largest have no mass in these integers and are never drawn.
#include "common.h"

namespace pa {
namespace smp {

constexpr int NT = 1024;

struct Args {
  const void* x;
  long long row;
  int V;
  const void* u;
  int u64;
  const float* t;
  const int* k;
  const float* p;
  const float* m;
  double t0, p0, m0;
  int k0;
  int64_t* ids;
  float* probs;
};

// order-preserving key of a logit; 0: not a token (NaN, -inf)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 -> +0: equal logits are ties
  const uint32_t k = (b >> 31) ? ~b : b | 0x80000000u;
  return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? k & 0x7fffffffu : ~k);
}

template <typename V>
__device__ __forceinline__ V wave_add(V v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// 2^y for y <= 0 by its Taylor series around the nearest integer, relative error under 10^-14; 0 under 2^-64
__device__ __forceinline__ double exp2_64(double y) {
  const double n = rint(y), f = (y - n) * 0.693147180559945309417;
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  const long long e = (long long)(y < -64.0 ? 0 : (int)n) << 52;
  return y >= -64.0 ? __builtin_bit_cast(double, __builtin_bit_cast(long long, p) + e) : 0.0;
}

// Weight of a logit beside the largest one: at most 1; 1 for every +inf and then 0 for the others
struct Weigh {
  double xm, s;  // largest logit, log2(e) / t
  __device__ __forceinline__ double operator()(float x) const {
    const double d = (double)x - xm;  // NaN for +inf beside +inf
    return d < 0.0 ? exp2_64(d * s) : 1.0;
  }
};

// Down to 10^-30 (0 and below: greedy), where log2(e) / t times a 32-bit logit is far from the 64-bit range's end
__device__ __forceinline__ double temperature(const Args& A, int r) {
  const double t = A.t ? (double)A.t[r] : A.t0;
  return t > 0.0 && t < 1e-30 ? 1e-30 : t;
}

struct Setting {
  double t, p, m, u;
  int k;
};
__device__ __forceinline__ Setting setting(const Args& A, int r) {
  Setting c;
  c.t = temperature(A, r);
  c.p = A.p ? (double)A.p[r] : A.p0;
  const double m = A.m ? (double)A.m[r] : A.m0, u = A.u64 ? reinterpret_cast<const double*>(A.u)[r]
                                                          : (double)reinterpret_cast<const float*>(A.u)[r];
  c.m = !(m > 0.0) ? 0.0 : (m < 1.0 ? m : 1.0);
  c.u = u >= 0.0 ? u : 0.0;  // 1 and above: the last kept token
  c.k = A.k ? A.k[r] : A.k0;
  return c;
}
constexpr double kLog2e = 1.44269504088896340736;

// A row by radix selection over keys, 8 bits a pass: thresholds by counts (k) and by masses (p).
template <typename T>
__device__ void radix_row(const Args& A, int r, uint32_t mk, uint32_t valid, const Setting& c_) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const int V = A.V, k = c_.k;
  const double p = c_.p, m = c_.m, u = c_.u;
  __shared__ uint32_t red[16];
  __shared__ uint32_t hist[256];
  __shared__ unsigned long long mass[256];
  __shared__ double dred[16];
  __shared__ uint32_t sk_, sc_;
  __shared__ unsigned long long sm_;
  const Weigh weigh{(double)value_of(mk), kLog2e / c_.t};
  auto weight = [&](uint32_t kk) -> double { return weigh(value_of(kk)); };
  const double fix = __builtin_ldexp(1.0, 62 - (32 - __builtin_clz(V)));
  auto fixed = [&](double w) -> unsigned long long { return (unsigned long long)(w * fix + 0.5); };

  // threshold key and how many of its ties are in the set: all tokens, then the first k
  uint32_t tk = 1, ck = 0xffffffffu;
  if (k > 0 && (uint32_t)k < valid) {
    uint32_t want = k, pre = 0;
    for (int s = 24; s >= 0; s -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t hi = s == 24 ? 0u : ~0u << (s + 8);
      for (int i = tid; i < V; i += NT) {
        const uint32_t kk = key_of(to_f(x[i]));
        if (kk != 0 && (kk & hi) == pre) atomicAdd(&hist[(kk >> s) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t w = want;
        int d = 255;
        for (; d > 0; --d) {
          if (hist[d] >= w) break;
          w -= hist[d];
        }
        sk_ = d;
        sc_ = w;
      }
      __syncthreads();
      pre |= sk_ << s;
      want = sc_;
      __syncthreads();
    }
    tk = pre;
    ck = want;
  }

  // mass of the set, and of it the part p
  if (p < 1.0) {
    if (!(p > 0.0)) {
      tk = mk;
      ck = 1;
    } else {
      uint32_t pre = 0;
      unsigned long long above = 0;
      double goal = 0.0;
      for (int s = 24; s >= 0; s -= 8) {
        if (tid < 256) mass[tid] = 0;
        __syncthreads();
        const uint32_t hi = s == 24 ? 0u : ~0u << (s + 8);
        for (int i = tid; i < V; i += NT) {
          const uint32_t kk = key_of(to_f(x[i]));
          if (kk > tk || (kk == tk && ck == 0xffffffffu && kk != 0))
            if ((kk & hi) == pre) atomicAdd(&mass[(kk >> s) & 255], fixed(weight(kk)));
        }
        __syncthreads();
        if (tid == 0 && ck != 0xffffffffu && (tk & hi) == pre) mass[(tk >> s) & 255] += ck * fixed(weight(tk));
        __syncthreads();
        if (s == 24) {
          unsigned long long all = 0;
          for (int i = 0; i < 256; ++i) all += mass[i];
          goal = p * (double)all;
        }
        if (tid == 0) {
          unsigned long long a = above;
          int d = 255, last = 255;
          for (; d >= 0; --d) {
            if (mass[d]) last = d;
            if ((double)(a + mass[d]) >= goal && mass[d]) break;
            if (d) a += mass[d];
          }
          if (d < 0) {  // rounding of the goal: the lowest that has any
            d = last;
            a = above;
            for (int j = 255; j > d; --j) a += mass[j];
          }
          sk_ = d;
          sm_ = a;
        }
        __syncthreads();
        pre |= sk_ << s;
        above = sm_;
        __syncthreads();
      }
      const double c = __builtin_ceil((goal - (double)above) / (double)fixed(weight(pre)));
      const uint32_t most = pre == tk ? ck : 0xffffffffu;
      ck = c < 1.0 ? 1u : (c < (double)most ? (uint32_t)c : most);
      tk = pre;
    }
  }

  // each wave's part of the row: kept mass above the threshold, and its ties
  const int span = ((V + 15) / 16 + 63) / 64 * 64, a0 = min(wave * span, V), a1 = min(a0 + span, V);
  const double wt = weight(tk);
  const bool tie_ok = wt >= m;
  double s = 0.0;
  uint32_t ties = 0;
  for (int i = a0 + lane; i < a1; i += 64) {
    const uint32_t kk = key_of(to_f(x[i]));
    if (kk > tk) {
      const double w = weight(kk);
      if (w >= m) s += w;
    } else if (kk == tk && kk != 0) {
      ++ties;
    }
  }
  s = wave_add(s);
  ties = wave_add(ties);
  if (lane == 0) { dred[wave] = s; red[wave] = ties; }
  __syncthreads();
  // with the waves before it, each wave's place in the kept mass
  double total = 0.0, before = 0.0;
  uint32_t seen = 0, seen_here = 0;
  for (int i = 0; i < 16; ++i) {
    if (i == wave) { before = total; seen_here = seen; }
    const uint32_t left = ck > seen ? ck - seen : 0, take = red[i] < left ? red[i] : left;
    total += dred[i] + (tie_ok ? take * wt : 0.0);  // one expression for all borders: they meet exactly
    seen += red[i];
  }
  const uint32_t left = ck > seen_here ? ck - seen_here : 0, take = red[wave] < left ? red[wave] : left;
  const double after = before + (dred[wave] + (tie_ok ? take * wt : 0.0)), goal = u * total;
  // the last wave whose part is not empty takes what rounding leaves over
  int lastw = 0;
  {
    uint32_t sn = 0;
    for (int i = 0; i < 16; ++i) {
      const uint32_t lf = ck > sn ? ck - sn : 0;
      if (dred[i] > 0.0 || (tie_ok && red[i] && lf)) lastw = i;
      sn += red[i];
    }
  }
  const bool mine = (goal >= before && goal < after) || (wave == lastw && goal >= total);
  if (!mine) return;
  int found = -1, final_kept = -1;
  double run = before, wf = 0.0, wl = 0.0;
  uint32_t tie = seen_here;
  for (int i0 = a0; i0 < a1 && found < 0; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t kk = i < a1 ? key_of(to_f(x[i])) : 0u;
    const bool is_tie = kk == tk && kk != 0;
    const unsigned long long tb = __ballot(is_tie);
    const uint32_t rank = tie + __popcll(tb & ((1ull << lane) - 1));
    tie += __popcll(tb);
    double w = 0.0;
    if (kk > tk) w = weight(kk);
    else if (is_tie && rank < ck) w = wt;
    if (!(w >= m)) w = 0.0;
    double c = w;  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double b = __shfl_up(c, o, 64);
      if (lane >= o) c += b;
    }
    const unsigned long long hit = __ballot(w > 0.0 && run + c > goal);
    const unsigned long long any = __ballot(w > 0.0);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      found = i0 + l;
      wf = __shfl(w, l, 64);
    } else if (any) {
      const int l = 63 - __builtin_clzll(any);
      final_kept = i0 + l;
      wl = __shfl(w, l, 64);
    }
    run += __shfl(c, 63, 64);
  }
  if (found < 0) { found = final_kept; wf = wl; }
  if (lane == 0) {
    A.ids[r] = found;
    A.probs[r] = (float)(wf / total);
  }
}

constexpr int CH = 8192;  // tokens of a chunk
constexpr int NB = 384;   // bins of 1/8 in log2 w: 47.9 octaves, and the last for what lies below
constexpr int CAP = NT;   // tokens of a border's bin that are ranked

struct Chunk {
  uint32_t key, valid, first, pad;  // largest key, tokens, lowest index of the largest
  uint32_t count[NB];
  unsigned long long mass[NB];      // relative to the chunk's largest logit, scaled by kFix
};
constexpr double kFix = 562949953421312.0;  // 2^49: 8192 tokens stay under 2^62

__device__ __forceinline__ double grid_of(float x, double s) { return floor((double)x * s * 8.0); }
// Bin of a logit under the largest one's place on the grid.  +inf: bin 0, and the last for what lies under it.
__device__ __forceinline__ int bin_of(float x, double s, double top) {
  const double d = top - grid_of(x, s);
  return d < (double)(NB - 1) ? (int)d : (d != d ? 0 : NB - 1);
}

// E consecutive tokens from i on; -inf past the end
template <typename T, int E>
__device__ __forceinline__ void load_tokens(const T* __restrict__ x, int i, int end, bool vec, float (&o)[E]) {
  if (vec && i + E <= end) {
    constexpr int W = 16 / sizeof(T) < E ? 16 / sizeof(T) : E;
#pragma unroll
    for (int j = 0; j < E; j += W) {
      float v[W];
      load_f<T, W>(x + i + j, v);
#pragma unroll
      for (int e = 0; e < W; ++e) o[j + e] = v[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = i + j < end ? to_f(x[i + j]) : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ bool vector_rows(const Args& A) {
  return (reinterpret_cast<uintptr_t>(A.x) & 15) == 0 && A.row % (16 / (int)sizeof(T)) == 0;
}

// What bounds it: the logits' read (once), beside about 20 64-bit operations and two LDS atomics a token.
template <typename T>
__global__ __launch_bounds__(256) void chunk_kernel(Args A, Chunk* __restrict__ out, int nc) {
  const int r = blockIdx.x / nc, ch = blockIdx.x % nc, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const int i0 = ch * CH, end = min(A.V, i0 + CH);
  Chunk* const C = out + blockIdx.x;
  __shared__ uint32_t rk[4], rv[4], ri[4];
  __shared__ uint32_t count[NB];
  __shared__ unsigned long long mass[NB];
  for (int i = tid; i < NB; i += 256) {
    count[i] = 0;
    mass[i] = 0;
  }
  constexpr int E = 8, P = CH / (256 * E);  // a thread's tokens: P times E in a row
  float v[P][E];
  const bool vec = vector_rows<T>(A);
  uint32_t mk = 0, mi = 0xffffffffu, valid = 0;
#pragma unroll
  for (int j = 0; j < P; ++j) load_tokens<T, E>(x, i0 + (j * 256 + tid) * E, end, vec, v[j]);
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t k = key_of(v[j][e]);
      valid += k != 0;
      if (k > mk) {
        mk = k;
        mi = i0 + (j * 256 + tid) * E + e;
      }
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t k = __shfl_xor(mk, o, 64), i = __shfl_xor(mi, o, 64);
    if (k > mk || (k == mk && i < mi)) {
      mk = k;
      mi = i;
    }
  }
  valid = wave_add(valid);
  if (lane == 0) {
    rk[wave] = mk;
    ri[wave] = mi;
    rv[wave] = valid;
  }
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    valid += rv[w];
    if (rk[w] > mk || (rk[w] == mk && ri[w] < mi)) {
      mk = rk[w];
      mi = ri[w];
    }
  }
  if (tid == 0) {
    C->key = mk;
    C->valid = valid;
    C->first = mi;
  }
  const double t = temperature(A, r);
  if (valid == 0 || !(t > 0.0)) return;  // no histogram is read
  const Weigh weigh{(double)value_of(mk), kLog2e / t};
  const double top = grid_of(value_of(mk), weigh.s);
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key_of(v[j][e]) != 0) {
        const int b = bin_of(v[j][e], weigh.s, top);
        atomicAdd(&count[b], 1u);
        if (b < NB - 1) atomicAdd(&mass[b], (unsigned long long)(weigh(v[j][e]) * kFix + 0.5));
      }
  __syncthreads();
  for (int i = tid; i < NB; i += 256) {
    C->count[i] = count[i];
    C->mass[i] = mass[i];
  }
}

// inclusive sums over the lanes
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V b = __shfl_up(v, o, 64);
    if (lane >= o) v += b;
  }
  return v;
}

// Bounded by latency: some ten dependent steps over a few KB, one re-read of the chunks that have a border's
// tokens, and one chunk's scan.
template <typename T>
__global__ __launch_bounds__(NT) void row_kernel(Args A, const Chunk* __restrict__ in, int nc) {
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const Chunk* const C = in + (long long)r * nc;
  __shared__ uint32_t rk[16], rv[16], ri[16];
  __shared__ uint32_t cum[NB];              // tokens up to and with a bin
  __shared__ double cmass[NB];              // and their mass
  __shared__ uint32_t lkey[CAP], lidx[CAP]; // tokens of a border's bin
  __shared__ unsigned long long lw[CAP];
  __shared__ uint32_t ln;
  __shared__ uint32_t tkey, tidx;           // the last kept token by top-k and top-p
  __shared__ double dsh, red[16];
  __shared__ int bsh;

  uint32_t mk = 0, mi = 0xffffffffu, valid = 0;
  for (int c = tid; c < nc; c += NT) {
    const uint32_t k = C[c].key, i = C[c].first;
    valid += C[c].valid;
    if (k > mk || (k == mk && i < mi)) {
      mk = k;
      mi = i;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t k = __shfl_xor(mk, o, 64), i = __shfl_xor(mi, o, 64);
    if (k > mk || (k == mk && i < mi)) {
      mk = k;
      mi = i;
    }
  }
  valid = wave_add(valid);
  if (lane == 0) {
    rk[wave] = mk;
    ri[wave] = mi;
    rv[wave] = valid;
  }
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    valid += rv[w];
    if (rk[w] > mk || (rk[w] == mk && ri[w] < mi)) {
      mk = rk[w];
      mi = ri[w];
    }
  }
  const Setting c_ = setting(A, r);
  if (valid == 0 || !(c_.t > 0.0)) {  // nothing to draw from, or the largest
    if (tid == 0) {
      A.ids[r] = valid == 0 ? -1 : (int64_t)mi;
      A.probs[r] = valid == 0 ? 0.f : 1.f;
    }
    return;
  }
  const Weigh weigh{(double)value_of(mk), kLog2e / c_.t};
  const double top = grid_of(value_of(mk), weigh.s);
  // a chunk's scale beside the row, and its bins' shift
  auto scale_of = [&](int c) -> double { return C[c].key ? weigh(value_of(C[c].key)) * (1.0 / kFix) : 0.0; };
  auto shift_of = [&](int c) -> int { return C[c].key ? bin_of(value_of(C[c].key), weigh.s, top) : NB; };
  auto fixed = [](double w) -> unsigned long long { return (unsigned long long)(w * kFix + 0.5); };

  // the chunks' histograms, joined; the last bin has what is left of the tokens, and no mass
  if (tid < NB) {
    uint32_t n = 0;
    double w = 0.0;
    if (tid < NB - 1)
      for (int c = 0; c < nc; ++c) {
        const int b = tid - shift_of(c);
        if (b >= 0) {
          n += C[c].count[b];
          w += (double)C[c].mass[b] * scale_of(c);
        }
      }
    cum[tid] = n;
    cmass[tid] = w;
  }
  __syncthreads();
  if (wave == 0) {
    constexpr int L = NB / 64;
    uint32_t n[L], ns = 0;
    double w[L], ws = 0.0;
#pragma unroll
    for (int j = 0; j < L; ++j) {
      n[j] = ns += cum[lane * L + j];
      w[j] = ws += cmass[lane * L + j];
    }
    const uint32_t nb = wave_scan(ns) - ns;
    const double wb = wave_scan(ws) - ws;
#pragma unroll
    for (int j = 0; j < L; ++j) {
      cum[lane * L + j] = nb + n[j];
      cmass[lane * L + j] = wb + w[j];
    }
  }
  __syncthreads();

  // Tokens of bin b into the list.  Their number is known; false where it does not fit.
  const bool vec = vector_rows<T>(A);
  int listed = -1;
  auto gather = [&](int b) -> bool {
    if (b == listed) return true;
    const uint32_t want = cum[b] - (b ? cum[b - 1] : 0u);
    if (want > CAP) return false;
    listed = b;
    __syncthreads();  // the list before has been read
    if (tid == 0) ln = 0;
    __syncthreads();
    for (int c = 0; c < nc; ++c) {
      const int lb = b - shift_of(c);
      if (lb < 0 || C[c].count[lb] == 0) continue;
      float v[8];
      load_tokens<T, 8>(x, c * CH + tid * 8, min(A.V, (c + 1) * CH), vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (key_of(v[e]) != 0 && bin_of(v[e], weigh.s, top) == b) {
          const uint32_t at = atomicAdd(&ln, 1u);
          if (at < CAP) {
            lkey[at] = key_of(v[e]);
            lidx[at] = c * CH + tid * 8 + e;
            lw[at] = fixed(weigh(v[e]));
          }
        }
    }
    __syncthreads();
    return true;
  };
  // of the list: tokens before this one in the order, and their mass (threads below ln)
  auto rank = [&](uint32_t& before, unsigned long long& mass) {
    const uint32_t n = ln;
    before = 0;
    mass = 0;
    if ((uint32_t)tid < n) {
      const uint32_t k = lkey[tid], i = lidx[tid];
      for (uint32_t j = 0; j < n; ++j)
        if (lkey[j] > k || (lkey[j] == k && lidx[j] < i)) {
          ++before;
          mass += lw[j];
        }
    }
  };

  // top-k: its last token, if it lies in a bin with mass, and the set's mass
  int bt = NB - 1;        // bin of the last kept token by top-k and top-p; NB - 1: no token with mass is cut
  bool ok = true;
  if (tid == 0) {
    tkey = 0;
    tidx = 0xffffffffu;
    dsh = cmass[NB - 1];
  }
  __syncthreads();
  if (c_.k > 0 && (uint32_t)c_.k < valid) {
    if (tid < NB - 1 && cum[tid] >= (uint32_t)c_.k && (tid == 0 || cum[tid - 1] < (uint32_t)c_.k)) rk[0] = tid;
    else if (tid == NB - 1 && cum[NB - 2] < (uint32_t)c_.k) rk[0] = NB - 1;
    __syncthreads();
    bt = (int)rk[0];
    if (bt < NB - 1) {
      ok = gather(bt);
      if (ok) {
        uint32_t before;
        unsigned long long mass;
        rank(before, mass);
        const uint32_t last = (uint32_t)c_.k - (bt ? cum[bt - 1] : 0u) - 1;  // its rank in the bin
        if ((uint32_t)tid < ln && before == last) {
          tkey = lkey[tid];
          tidx = lidx[tid];
          dsh = (bt ? cmass[bt - 1] : 0.0) + (double)(mass + lw[tid]) * (1.0 / kFix);
        }
      }
    }
    __syncthreads();
  }
  // top-p within it
  if (ok && c_.p < 1.0) {
    if (!(c_.p > 0.0)) {  // the first token alone
      if (tid == 0) {
        tkey = mk;
        tidx = mi;
      }
      bt = 0;
      __syncthreads();
    } else {
      const double goal = c_.p * dsh;
      const int bk = bt;
      if (tid == 0) bsh = NB - 1;
      __syncthreads();
      // the first bin whose tokens take the mass to the goal; at or behind top-k's own: that one
      if (tid < NB && cmass[tid] >= goal && (tid == 0 || cmass[tid - 1] < goal)) bsh = tid;
      __syncthreads();
      const int bp = min(bsh, bk);
      if (bp < NB - 1) {
        ok = gather(bp);
        if (ok) {
          uint32_t before;
          unsigned long long mass;
          rank(before, mass);
          const double above = bp ? cmass[bp - 1] : 0.0;
          // kept: less than the goal lies before it, and top-k has it
          const bool in = (uint32_t)tid < ln && (lkey[tid] > tkey || (lkey[tid] == tkey && lidx[tid] <= tidx));
          const bool kept = in && (above + (double)mass * (1.0 / kFix) < goal || (bp == 0 && before == 0));
          // the last of them: the one with the most before it
          uint32_t best = kept ? before + 1 : 0;
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) best = max(best, (uint32_t)__shfl_xor(best, o, 64));
          if (lane == 0) rk[wave] = best;
          __syncthreads();
          best = 0;
#pragma unroll
          for (int w = 0; w < 16; ++w) best = max(best, rk[w]);
          // (rounding: none of this bin's, then all of the bins above, whose last token is not looked for)
          if (best == 0) {
            if (tid == 0) {
              tkey = 0xffffffffu;
              tidx = 0;
            }
          } else if (kept && before + 1 == best) {
            tkey = lkey[tid];
            tidx = lidx[tid];
          }
          bt = bp;
          __syncthreads();
        }
      }
    }
  }
  if (!ok) {
    radix_row<T>(A, r, mk, valid, c_);
    return;
  }
  // min-p: the bin of its border
  int bf = bt;
  if (c_.m > 0.0) {
    const double ym = (double)value_of(mk) * weigh.s + log2(c_.m), d = top - floor(ym * 8.0);
    const int bm = d < (double)(NB - 1) ? max((int)d, 0) : (d != d ? 0 : NB - 1);
    if (bm < bf) bf = bm;
  }
  // bins before bf are kept whole, of bf what passes the tests, nothing behind it
  const uint32_t tk = tkey, ti = tidx;
  auto passes = [&](uint32_t k, uint32_t i, double w) { return (k > tk || (k == tk && i <= ti)) && w >= c_.m; };
  __shared__ unsigned long long fsh;
  const bool partial = bf < NB - 1;
  if (partial) {
    if (!gather(bf)) {
      radix_row<T>(A, r, mk, valid, c_);
      return;
    }
    if (tid == 0) fsh = 0;
    __syncthreads();
    unsigned long long w = 0;
    if ((uint32_t)tid < ln) w = passes(lkey[tid], lidx[tid], weigh(value_of(lkey[tid]))) ? lw[tid] : 0;
    w = wave_add(w);
    if (lane == 0 && w) atomicAdd(&fsh, w);
    __syncthreads();
  }
  const double whole = bf > 0 ? cmass[bf - 1] : 0.0, total = whole + (partial ? (double)fsh * (1.0 / kFix) : 0.0);
  const double goal = c_.u * total;

  // the chunk in which the kept mass passes the goal: one wave sums a chunk's whole bins and its listed tokens
  double run = 0.0, start = 0.0;
  int at = -1, lastc = -1;
  double lastrun = 0.0;
  for (int c0 = 0; c0 < nc && at < 0; c0 += 16) {
    const int c = c0 + wave;
    double w = 0.0;
    if (c < nc) {
      const int hi = min(bf - shift_of(c), NB - 1);
      for (int b = lane; b < hi; b += 64) w += (double)C[c].mass[b];
      w *= scale_of(c);
      if (partial) {
        unsigned long long f = 0;
        for (uint32_t j = lane; j < ln; j += 64)
          if (lidx[j] / CH == (uint32_t)c && passes(lkey[j], lidx[j], weigh(value_of(lkey[j])))) f += lw[j];
        w += (double)f * (1.0 / kFix);
      }
      w = wave_add(w);
    }
    __syncthreads();
    if (lane == 0) red[wave] = w;
    __syncthreads();
    for (int j = 0; j < 16 && c0 + j < nc; ++j) {
      const double q = red[j];
      if (q > 0.0) {
        lastc = c0 + j;
        lastrun = run;
        if (run + q > goal) {
          at = c0 + j;
          start = run;
          break;
        }
      }
      run += q;
    }
  }
  if (at < 0) {  // rounding: the last chunk that has any
    at = lastc;
    start = lastrun;
  }
  // scan of that chunk, 8 tokens a thread
  float v[8];
  double w[8], sum = 0.0;
  load_tokens<T, 8>(x, at * CH + tid * 8, min(A.V, (at + 1) * CH), vec, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t k = key_of(v[e]);
    w[e] = 0.0;
    if (k != 0) {
      const int b = bin_of(v[e], weigh.s, top);
      if (b < bf || (partial && b == bf)) {
        const double q = weigh(v[e]);
        if (b < bf || passes(k, at * CH + tid * 8 + e, q)) w[e] = q;
      }
    }
    sum += w[e];
  }
  const double inc = wave_scan(sum);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  if (tid == 0) {
    rk[0] = 0xffffffffu;  // lowest index that passes the goal
    rv[0] = 0;            // 1 + the last token with mass
  }
  __syncthreads();
  double before = start + inc - sum;
  for (int j = 0; j < wave; ++j) before += red[j];
  uint32_t hit = 0xffffffffu, last = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    before += w[e];
    if (w[e] > 0.0) {
      last = tid * 8 + e + 1;
      if (before > goal && hit == 0xffffffffu) hit = tid * 8 + e;
    }
  }
  if (hit != 0xffffffffu) atomicMin(&rk[0], hit);
  if (last) atomicMax(&rv[0], last);
  __syncthreads();
  const uint32_t found = rk[0] != 0xffffffffu ? rk[0] : rv[0] - 1;  // rounding: the last with mass
  if ((uint32_t)tid == found / 8) {
    double q = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((uint32_t)e == found % 8) q = w[e];
    A.ids[r] = (int64_t)at * CH + found;
    A.probs[r] = (float)(q / total);
  }
}

}  // namespace smp
}  // namespace pa

// x: [rows, V] logits (row stride in elements); u: [rows] in [0, 1) (fp32 or fp64); t / k / p / m: [rows] or
// null for the scalars beside them.  ids int64 [rows], probs fp32 [rows] (share of the kept mass).
// ws: rows * pa_sample_ws_bytes(V) bytes, 8-byte aligned.
PA_API long long pa_sample_ws_bytes(int V) {
  return (long long)((V + pa::smp::CH - 1) / pa::smp::CH) * (long long)sizeof(pa::smp::Chunk);
}

PA_API int pa_sample(const void* x, long long row, int rows, int V, const void* u, int u64, const float* t,
                     const int* k, const float* p, const float* m, double t0, int k0, double p0, double m0,
                     int64_t* ids, float* probs, void* ws, int dt, hipStream_t st) {
  if (rows == 0) return 0;
  if (rows < 0 || V <= 0 || V > (1 << 30) || !u || !ids || !probs || !ws) return (int)hipErrorInvalidValue;
  pa::smp::Args A{x, row, V, u, u64, t, k, p, m, t0, p0, m0, k0, ids, probs};
  const int nc = (V + pa::smp::CH - 1) / pa::smp::CH;
  if (rows * (long long)nc > 0x7fffffff) return (int)hipErrorInvalidValue;
  pa::smp::Chunk* C = (pa::smp::Chunk*)ws;
  PA_DISPATCH_DTYPE(dt, T, {
    pa::smp::chunk_kernel<T><<<(int)(rows * (long long)nc), 256, 0, st>>>(A, C, nc);
    pa::smp::row_kernel<T><<<rows, pa::smp::NT, 0, st>>>(A, C, nc);
  })
  return (int)hipGetLastError();
}
