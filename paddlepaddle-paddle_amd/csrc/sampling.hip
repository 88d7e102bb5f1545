// Sampling of one token per row from filtered logits with given random numbers.
//
// Mathematics.  w_i = exp((x_i - max x) / t).  The kept set is, of the tokens in the order of falling x
// (equal x: the lower index first), the first k; of those the ones before which less than p of their mass
// lies (at least one); of those the ones with w_i >= m.  The answer is the first token, in the order of the
// vocabulary, at which the kept mass passes u times its total.  Tokens of -inf or NaN are never kept.
//
// No sort: the kept set is "x above a threshold, and of the x equal to it the first c", and both thresholds
// are found by radix selection over order-preserving 32-bit keys, on counts (k) and on masses (p).
// Histograms of masses are 64-bit integers (w scaled by 2^S with S so large that a row's sum just fits), so
// their atomics add exactly and the answer does not depend on their order; weights and sums are 64-bit
// floats, since a 32-bit sum over 10^5 tokens moves the borders of the cumulative distribution by more than
// a token's share.
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

template <typename T>
__global__ __launch_bounds__(NT) void sample_kernel(Args A) {
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const int V = A.V;
  __shared__ uint32_t red[16];
  __shared__ uint32_t hist[256];
  __shared__ unsigned long long mass[256];
  __shared__ double dred[16];
  __shared__ uint32_t sk_, sc_;
  __shared__ unsigned long long sm_;

  // maximum, and the number of tokens
  uint32_t mk = 0, valid = 0;
  for (int i = tid; i < V; i += NT) {
    const uint32_t k = key_of(to_f(x[i]));
    mk = k > mk ? k : mk;
    valid += k != 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t b = __shfl_xor(mk, o, 64);
    mk = b > mk ? b : mk;
  }
  valid = wave_add(valid);
  if (lane == 0) { red[wave] = mk; hist[wave] = valid; }
  __syncthreads();
  valid = 0;
  for (int i = 0; i < 16; ++i) { mk = red[i] > mk ? red[i] : mk; valid += hist[i]; }
  __syncthreads();
  if (valid == 0) {
    if (tid == 0) { A.ids[r] = -1; A.probs[r] = 0.f; }
    return;
  }
  const double t = A.t ? (double)A.t[r] : A.t0, p = A.p ? (double)A.p[r] : A.p0;
  const double m_in = A.m ? (double)A.m[r] : A.m0, m = !(m_in > 0.0) ? 0.0 : (m_in < 1.0 ? m_in : 1.0);
  const int k = A.k ? A.k[r] : A.k0;
  const double u_in = A.u64 ? reinterpret_cast<const double*>(A.u)[r] : (double)reinterpret_cast<const float*>(A.u)[r];
  const double u = u_in >= 0.0 ? u_in : 0.0;  // 1 and above: the last kept token
  if (!(t > 0.0)) {  // greedy
    uint32_t best = 0xffffffffu;
    for (int i = tid; i < V; i += NT)
      if (key_of(to_f(x[i])) == mk && (uint32_t)i < best) best = i;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint32_t b = __shfl_xor(best, o, 64);
      best = b < best ? b : best;
    }
    if (lane == 0) red[wave] = best;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < 16; ++i) best = red[i] < best ? red[i] : best;
      A.ids[r] = best;
      A.probs[r] = 1.f;
    }
    return;
  }
  const double xm = (double)value_of(mk), it = 1.0 / t;
  auto weight = [&](uint32_t kk) -> double { return kk == mk ? 1.0 : exp(((double)value_of(kk) - xm) * it); };
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

}  // namespace smp
}  // namespace pa

// x: [rows, V] logits (row stride in elements); u: [rows] in [0, 1) (fp32 or fp64); t / k / p / m: [rows] or
// null for the scalars beside them.  ids int64 [rows], probs fp32 [rows] (share of the kept mass).
PA_API int pa_sample(const void* x, long long row, int rows, int V, const void* u, int u64, const float* t,
                     const int* k, const float* p, const float* m, double t0, int k0, double p0, double m0,
                     int64_t* ids, float* probs, int dt, hipStream_t st) {
  if (rows == 0) return 0;
  if (rows < 0 || V <= 0 || !u || !ids || !probs) return (int)hipErrorInvalidValue;
  pa::smp::Args A{x, row, V, u, u64, t, k, p, m, t0, p0, m0, k0, ids, probs};
  PA_DISPATCH_DTYPE(dt, T, pa::smp::sample_kernel<T><<<rows, pa::smp::NT, 0, st>>>(A))
  return (int)hipGetLastError();
}
