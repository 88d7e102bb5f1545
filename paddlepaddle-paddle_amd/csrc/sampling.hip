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
// by more than a token's share.  Masses that are added by atomics are 64-bit integers (a bin's in units of 2^-48 of its
// upper end, a listed token's in 2^-49 of the largest), so the answer does not depend on their order.  Tokens under
// 2^-47 of the largest lie in the last bin, which has no mass, and are never drawn.
#include "common.h"

namespace pa {
namespace smp {

constexpr int NT = 512;       // threads of a row's block
constexpr int NW = NT / 64;

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
  int k0, own;  // own: bits 0 .. 3, whether t, k, p, m are arrays (else they point to memory that may be read)
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

// Lane exchanges by DPP (no trip through LDS): the value of another lane, or 0 where there is none
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V from_lane(V v) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
  } else {
    struct Two {
      int a, b;
    };
    Two t = __builtin_bit_cast(Two, v);
    t.a = __builtin_amdgcn_update_dpp(0, t.a, CTRL, ROWS, 0xf, true);
    t.b = __builtin_amdgcn_update_dpp(0, t.b, CTRL, ROWS, 0xf, true);
    return __builtin_bit_cast(V, t);
  }
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int lane) {  // of a lane that all lanes name
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    struct Two {
      int a, b;
    };
    Two t = __builtin_bit_cast(Two, v);
    t.a = __builtin_amdgcn_readlane(t.a, lane);
    t.b = __builtin_amdgcn_readlane(t.b, lane);
    return __builtin_bit_cast(V, t);
  }
}
// Inclusive sums over the lanes: shifts by 1, 2, 4, 8 within rows of 16, then the rows' ends to the rows behind
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  v += from_lane<0x111, 0xf>(v);
  v += from_lane<0x112, 0xf>(v);
  v += from_lane<0x114, 0xf>(v);
  v += from_lane<0x118, 0xf>(v);
  v += from_lane<0x142, 0xa>(v);
  v += from_lane<0x143, 0xc>(v);
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_add(V v) {
  return lane_value(wave_scan(v), 63);
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = max(v, from_lane<0x111, 0xf>(v));
  v = max(v, from_lane<0x112, 0xf>(v));
  v = max(v, from_lane<0x114, 0xf>(v));
  v = max(v, from_lane<0x118, 0xf>(v));
  v = max(v, from_lane<0x142, 0xa>(v));
  v = max(v, from_lane<0x143, 0xc>(v));
  return lane_value(v, 63);
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
  const double v = (double)A.t[r], t = A.own & 1 ? v : A.t0;
  return t > 0.0 && t < 1e-30 ? 1e-30 : t;
}

struct Setting {
  double t, p, m, u;
  int k;
};
// (all loads at once: a branch for each setting would wait for them one by one)
__device__ __forceinline__ Setting setting(const Args& A, int r) {
  const float p = A.p[r], m_ = A.m[r], u32 = reinterpret_cast<const float*>(A.u)[A.u64 ? 2 * r : r],
              u32b = reinterpret_cast<const float*>(A.u)[A.u64 ? 2 * r + 1 : r];
  const int k = A.k[r];
  Setting c;
  c.t = temperature(A, r);
  const double p_ = A.own & 4 ? (double)p : A.p0;
  c.p = p_ > 0.0 ? p_ : 0.0;  // (NaN: the first token alone)
  const double m = A.own & 8 ? (double)m_ : A.m0;
  const uint64_t w = (uint64_t)__builtin_bit_cast(uint32_t, u32b) << 32 | __builtin_bit_cast(uint32_t, u32);
  const double u = A.u64 ? __builtin_bit_cast(double, w) : (double)u32;
  c.m = !(m > 0.0) ? 0.0 : (m < 1.0 ? m : 1.0);
  c.u = u >= 0.0 ? u : 0.0;  // 1 and above: the last kept token
  c.k = A.own & 2 ? k : A.k0;
  return c;
}
constexpr double kLog2e = 1.44269504088896340736;

// A row by radix selection over keys, 8 bits a pass: thresholds by counts (k) and by masses (p).
template <typename T>
__device__ __attribute__((noinline)) void radix_row(const Args& A, int r, uint32_t mk, uint32_t valid, const Setting& c_) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const int V = A.V, k = c_.k;
  const double p = c_.p, m = c_.m, u = c_.u;
  __shared__ uint32_t red[NW];
  __shared__ uint32_t hist[256];
  __shared__ unsigned long long mass[256];
  __shared__ double dred[NW];
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
  const int span = ((V + NW - 1) / NW + 63) / 64 * 64, a0 = min(wave * span, V), a1 = min(a0 + span, V);
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
  for (int i = 0; i < NW; ++i) {
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
    for (int i = 0; i < NW; ++i) {
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
constexpr int CAP = 1024; // tokens of a border's bin that are listed
constexpr int MC = 64;    // chunks whose scales are held at a time
constexpr int WITH = 1024;  // parts that are looked through at a time

constexpr int SUB = 128;  // tokens of a part of a chunk: 16 lanes' 8 each
struct Chunk {
  uint32_t key, valid, first, pad;  // largest key, tokens, lowest index of the largest
  uint32_t part[CH / SUB];          // largest key of each part
  uint32_t count[NB];
  unsigned long long mass[NB];      // sums of part_mass()
};
// A logit on the grid of 1/8 in log2 w: 8 log2 w = (place on the grid) + f, 0 <= f <= 1.  Bin: places under the largest
// logit's.  +inf: bin 0, f 0, and the last bin for what lies under it.
struct Grid {
  double s8, top;
  __device__ __forceinline__ int bin(float x, double& f) const {
    const double g = floor((double)x * s8), d = top - g;
    // (written out: the same weight wherever it is computed; NaN, of infinities: 0; places from 2^53 on: any of [0, 1])
    f = fmin(fmax(fma((double)x, s8, -g), 0.0), 1.0);
    int b;
    asm("v_cvt_i32_f64 %0, %1" : "=v"(b) : "v"(d));  // NaN: 0; beyond the integers: the largest
    return min(b, NB - 1);
  }
  __device__ __forceinline__ int bin(float x) const {
    double f;
    return bin(x, f);
  }
};
__device__ __forceinline__ Grid grid_of(uint32_t key, double t) {
  Grid g;
  g.s8 = 8.0 * kLog2e / t;
  const double x = (double)value_of(key);
  g.top = x < INFINITY ? floor(x * g.s8) : INFINITY;  // (also where s8 is 0)
  return g;
}
// 2^(f / 8) scaled by 2^48, plus `more`: its Taylor polynomial around the middle (relative error under 10^-13), multiplied
// out to powers of f
constexpr double kPart = 281474976710656.0;
struct Powers {
  double c[7];
  constexpr Powers() : c{} {
    const double a = 0.0866433975699931636771;      // ln 2 / 8
    double t = 1.0442737824274138403 * kPart;       // 2^(1 / 16) a^k / k!
    for (int k = 0; k < 7; ++k, t *= a / k) {
      double w = t;                                 // of (f - 1/2)^k: binomial(k, j) (-1/2)^(k - j) f^j
      for (int j = k; j >= 0; --j) {
        c[j] += w;
        w *= -0.5 * j / (k - j + 1);
      }
    }
  }
};
__device__ __forceinline__ double part(double f, double more) {
  constexpr Powers P;
  double p = P.c[6];
  p = fma(p, f, P.c[5]);
  p = fma(p, f, P.c[4]);
  p = fma(p, f, P.c[3]);
  p = fma(p, f, P.c[2]);
  p = fma(p, f, P.c[1]);
  return fma(p, f, P.c[0] + more);
}
// rounded: what a token adds to its bin's mass
__device__ __forceinline__ unsigned long long part_mass(double f) {
  return __builtin_bit_cast(unsigned long long, part(f, 4503599627370496.0)) & 0xfffffffffffffull;  // (on 2^52, whose last place is 1)
}
// a token's weight, with 1 at the upper end of bin 0; scale: of the bins' masses
__device__ __forceinline__ double weight(const Grid& G, const double* scale, float x) {
  double f;
  const int b = G.bin(x, f);
  return part(f, 0.0) * scale[b];
}
// w scaled by 2^49 and rounded, for w in [0, 1]: a listed token's mass
constexpr double kFix = 562949953421312.0;
__device__ __forceinline__ unsigned long long fixed(double w) {
  return __builtin_bit_cast(unsigned long long, fma(w, kFix, 4503599627370496.0)) & 0xfffffffffffffull;
}
// The least key whose logit's bin is b or before it.  By a whole wave, 6 bits a step.
__device__ __forceinline__ uint32_t least_key(const Grid& G, int b) {
  const uint32_t lane = threadIdx.x & 63, top = key_of(INFINITY);
  uint32_t key = 0;  // (0: no token's)
#pragma unroll 1
  for (int sh = 26; sh >= -4; sh -= 6) {
    const uint32_t step = sh >= 0 ? lane << sh : lane >> 4, k = key + step;  // (the last step: its 4 keys, 16 times each)
    const float v = value_of(k);
    const bool in = k >= top || (v > -INFINITY && G.bin(v) <= b);
    const int before = __popcll(__ballot(!in));
    if (before == 0) break;
    key += sh >= 0 ? (uint32_t)(before - 1) << sh : (uint32_t)before >> 4;
  }
  return key;
}
// a token's place in the order: larger ones come first
__device__ __forceinline__ unsigned long long place(uint32_t key, uint32_t i) {
  return (unsigned long long)key << 32 | (0xffffffffu - i);
}

// E consecutive tokens from i on; -inf past the end
template <typename T, int E>
__device__ __forceinline__ void load_tokens(const T* __restrict__ x, int i, int end, bool vec, T (&o)[E]) {
  if (vec && i + E <= end) {
    constexpr int W = 16 / sizeof(T) < E ? 16 / sizeof(T) : E;
#pragma unroll
    for (int j = 0; j < E; j += W) {
      const Pack<T, W> v = *reinterpret_cast<const Pack<T, W>*>(x + i + j);
#pragma unroll
      for (int e = 0; e < W; ++e) o[j + e] = v.v[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = i + j < end ? x[i + j] : from_f<T>(-INFINITY);
  }
}
template <typename T>
__device__ __forceinline__ bool vector_rows(const Args& A) {
  return (reinterpret_cast<uintptr_t>(A.x) & 15) == 0 && A.row % (16 / (int)sizeof(T)) == 0;
}

// What bounds it: vector instructions, 38 a token of which some 13 are 64-bit (a 32-bit mass would move the borders): their
// issue takes half of the time; the LDS a fifth, more than half of that in bank conflicts of the bins.  64 rows of 128256
// tokens in bf16 17 us, 512 rows of 32000 in fp32 27 us (2.4 TB/s), one row of 50304 8 us.  With one atomic for count and
// mass instead of two, and with four copies of the bins, a twentieth less.  Lists of a chunk's largest 128 tokens, written
// here, save the row's block 16 of 50 us at 128256 tokens and cost 6 here, and at 32000 they cost 8 and save none: the
// row's block looks the tokens up by the maxima of parts at every size.
template <typename T>
__global__ __launch_bounds__(256) void chunk_kernel(Args A, Chunk* __restrict__ out, int nc) {
  const int r = blockIdx.x / nc, ch = blockIdx.x % nc, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const int i0 = ch * CH, end = min(A.V, i0 + CH);
  Chunk* const C = out + blockIdx.x;
  __shared__ uint32_t rk[CH / SUB], rv, ri;
  __shared__ uint32_t count[NB];
  __shared__ unsigned long long mass[NB];
  for (int i = tid; i < NB; i += 256) {
    count[i] = 0;
    mass[i] = 0;
  }
  if (tid == 0) {
    rv = 0;
    ri = 0xffffffffu;
  }
  constexpr int E = 8, P = CH / (256 * E);  // a thread's tokens: P times E in a row, a wave's: P parts
  static_assert(SUB == 16 * E && CH / SUB == 64, "a part is 16 lanes', a chunk's parts a wave's lanes");
  T v[P][E];
  const bool vec = vector_rows<T>(A);
  uint32_t valid = 0;
#pragma unroll
  for (int j = 0; j < P; ++j) load_tokens<T, E>(x, i0 + (j * 256 + tid) * E, end, vec, v[j]);
  __syncthreads();
  uint32_t most[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t k = key_of(to_f(v[j][e]));
      valid += k != 0;
      m = max(m, k);
    }
    most[j] = m;
    m = max(m, from_lane<0x111, 0xf>(m));  // over the 16 lanes, in the last of them
    m = max(m, from_lane<0x112, 0xf>(m));
    m = max(m, from_lane<0x114, 0xf>(m));
    m = max(m, from_lane<0x118, 0xf>(m));
    if ((lane & 15) == 15) {
      rk[j * 16 + (tid >> 4)] = m;
      C->part[j * 16 + (tid >> 4)] = m;
    }
  }
  valid = wave_add(valid);
  if (lane == 0) atomicAdd(&rv, valid);
  __syncthreads();
  valid = rv;
  const uint32_t mk = wave_max_u(rk[lane]);
#pragma unroll
  for (int j = 0; j < P; ++j)
    if (most[j] == mk && mk != 0) {  // the thread has it
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (key_of(to_f(v[j][e])) == mk) atomicMin(&ri, (uint32_t)(i0 + (j * 256 + tid) * E + e));
    }
  __syncthreads();
  if (tid == 0) {
    C->key = mk;
    C->valid = valid;
    C->first = ri;
  }
  const double t = temperature(A, r);
  if (valid == 0 || !(t > 0.0)) return;  // no histogram is read
  const Grid G = grid_of(mk, t);
  // Rolled, the tokens read again from the caches: at one block a CU the code's own way into the instruction cache is
  // what takes longest
#pragma unroll 1
  for (int j = 0; j < P; ++j) {
    T q[E];
    load_tokens<T, E>(x, i0 + (j * 256 + tid) * E, end, vec, q);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key_of(to_f(q[e])) != 0) {
        double f;
        const int b = G.bin(to_f(q[e]), f);
        atomicAdd(&count[b], 1u);
        atomicAdd(&mass[b], part_mass(f));
      }
  }
  __syncthreads();
  for (int i = tid; i < NB; i += 256) {
    C->count[i] = count[i];
    C->mass[i] = mass[i];
  }
}

// Bounded by latency: some ten dependent steps over a few KB, one re-read of the parts that have a border's tokens, and
// one chunk's scan.  One row of 50304 tokens 18 us (4 the first loads, 3 the join of the histograms, 5 the list, 1 each
// selection); 64 rows of 128256 37 .. 45 us, as their longest list is; 512 rows of 32000 40 .. 43 us.
template <typename T>
__global__ __launch_bounds__(NT, 4) void row_kernel(Args A, const Chunk* __restrict__ in, int nc) {
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ x = reinterpret_cast<const T*>(A.x) + (long long)r * A.row;
  const Chunk* const C = in + (long long)r * nc;
  struct Token {
    unsigned long long place, w;              // w: fixed(), 0 once it is not kept
  };
  __shared__ uint32_t rk[NW], rv[NW], ri[NW];
  __shared__ uint32_t cum[NB];                // tokens up to and with a bin
  __shared__ double cmass[NB];                // and their mass
  __shared__ Token list[CAP];                 // tokens of a border's bin
  __shared__ uint32_t ln;                     // their number
  __shared__ uint32_t pcount[256];
  __shared__ unsigned long long pmass[256], fsh;
  __shared__ double red[NW], scale[NB];
  __shared__ uint32_t kmax, kmin;             // their keys
  __shared__ int bsh, shift[MC], with[WITH], wn;
  __shared__ unsigned long long got[2];

  uint32_t mk = 0, mi = 0xffffffffu, valid = 0;
  if (tid < nc) {
    mk = C[tid].key;
    mi = C[tid].first;
    valid = C[tid].valid;
  }
  const uint32_t own_key = mk;
  const Setting S = setting(A, r);
  for (int c = tid + NT; c < nc; c += NT) {
    const uint32_t k = C[c].key, i = C[c].first;
    valid += C[c].valid;
    if (k > mk || (k == mk && i < mi)) {
      mk = k;
      mi = i;
    }
  }
  valid = wave_add(valid);
  {
    const uint32_t k = wave_max_u(mk);
    mi = ~wave_max_u(mk == k ? ~mi : 0u);  // its lowest index
    mk = k;
  }
  if (lane == 0) {
    rk[wave] = mk;
    ri[wave] = mi;
    rv[wave] = valid;
  }
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    valid += rv[w];
    if (rk[w] > mk || (rk[w] == mk && ri[w] < mi)) {
      mk = rk[w];
      mi = ri[w];
    }
  }
  if (valid == 0 || !(S.t > 0.0)) {  // nothing to draw from, or the largest
    if (tid == 0) {
      A.ids[r] = valid == 0 ? -1 : (int64_t)mi;
      A.probs[r] = valid == 0 ? 0.f : 1.f;
    }
    return;
  }
  const Grid G = grid_of(mk, S.t);
  // the shifts of the bins of chunks [c0, c0 + MC)
  auto shifts = [&](int c0) {
    __syncthreads();
    if (tid < MC && c0 + tid < nc) {
      const uint32_t k = c0 ? C[c0 + tid].key : own_key;
      shift[tid] = k ? G.bin(value_of(k)) : NB;
    }
    __syncthreads();
  };
  if (tid < NB) scale[tid] = exp2_64(-0.125 * (double)(tid + 1)) * (1.0 / kPart);  // of a bin's mass

  // the chunks' histograms, joined; the last bin has no mass
  {
    uint32_t n = 0;
    double w = 0.0;
    for (int c0 = 0; c0 < nc; c0 += MC) {
      shifts(c0);
      if (tid < NB - 1) {
        const int e = min(MC, nc - c0);
#pragma unroll 16
        for (int c = 0; c < e; ++c) {
          const int b = tid - shift[c], at = max(b, 0);
          const uint32_t cn = C[c0 + c].count[at];
          const double cw = (double)C[c0 + c].mass[at];
          n += b >= 0 ? cn : 0u;
          w += b >= 0 ? cw : 0.0;
        }
      }
    }
    if (tid < NB) {
      cum[tid] = n;
      cmass[tid] = w * scale[tid];
    }
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

  // Tokens of bins [b0, b1] into the list.  Their number is known; false where it does not fit.  The parts of the row
  // whose largest token lies before b0's end are read, 16 tokens a lane and two parts a wave at a time.
  const bool vec = vector_rows<T>(A);
  int listed = -1;
  auto gather = [&](int b0, int b1) -> bool {
    if (b1 == listed) return true;
    if (cum[b1] - (b0 ? cum[b0 - 1] : 0u) > CAP) return false;
    listed = b1;
    constexpr int PP = CH / SUB;
    // their logits: [from, upto)
    const float from = value_of(least_key(G, b1)), upto = b0 ? value_of(least_key(G, b0 - 1)) : INFINITY;
    __syncthreads();  // the list before has been read
    if (tid == 0) {
      ln = 0;
      kmax = 0;
      kmin = 0xffffffffu;
    }
    for (int p0 = 0; p0 < nc * PP; p0 += WITH) {
      if (tid == 0) wn = 0;
      __syncthreads();
      for (int p = p0 + tid; p - tid < min(p0 + WITH, nc * PP); p += NT) {
        const uint32_t k = p < nc * PP ? C[p / PP].part[p % PP] : 0;
        const unsigned long long in = __ballot(k != 0 && value_of(k) >= from);
        int at = 0;
        if (lane == 0) at = atomicAdd(&wn, __popcll(in));
        at = lane_value(at, 0) + __popcll(in & ((1ull << lane) - 1));
        if (in >> lane & 1) with[at] = p;
      }
      __syncthreads();
      const int n = wn;
      // PF times 4 parts of a wave are on their way at once: as many bytes as its registers take
      constexpr int PF = sizeof(T) == 2 ? 4 : 2;
#pragma unroll 1
      for (int g = 4 * wave; g < n; g += 4 * PF * NW) {
        T raw[PF][8];
        int first[PF];
#pragma unroll
        for (int k = 0; k < PF; ++k) {
          const int j = g + 4 * k * NW + (lane >> 4);
          first[k] = j < n ? with[j] * SUB + (lane & 15) * 8 : A.V;
          load_tokens<T, 8>(x, first[k], A.V, vec, raw[k]);
        }
        auto in = [&](int k, int e) {
          const float v = to_f(raw[k][e]);
          return v >= from && (b0 == 0 || v < upto);
        };
        int own = 0;
#pragma unroll
        for (int k = 0; k < PF; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) own += in(k, e);
        const int before = wave_scan(own), all = lane_value(before, 63);
        if (all == 0) continue;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&ln, (uint32_t)all);
        at = lane_value(at, 0) + before - own;
#pragma unroll
        for (int k = 0; k < PF; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (in(k, e)) {
              if (at < CAP) list[at].place = first[k] + e;
              ++at;
            }
      }
      __syncthreads();
    }
    if (ln != cum[b1] - (b0 ? cum[b0 - 1] : 0u)) return false;  // (not seen; what follows relies on it)
    uint32_t hi = 0, lo = 0xffffffffu;
    for (uint32_t i = tid; i < ln; i += NT) {
      const uint32_t id = (uint32_t)list[i].place, k = key_of(to_f(x[id]));
      list[i] = Token{place(k, id), fixed(weight(G, scale, value_of(k)))};
      hi = max(hi, k);
      lo = min(lo, k);
    }
    hi = wave_max_u(hi);
    lo = ~wave_max_u(~lo);
    if (lane == 0 && hi) {
      atomicMax(&kmax, hi);
      atomicMin(&kmin, lo);
    }
    __syncthreads();
    return true;
  };
  // Of the listed tokens that are kept, in the order of falling places (or rising indexes, BY_INDEX): by count, the one
  // with `last` before it; by mass, the last one before which less than `room` lies.  `at`: its place; `mass`: up to and
  // with it.  The range of the order that holds it is cut into 256 parts until few tokens are left to be ranked.
  auto select = [&](bool by_index, bool by_mass, uint32_t last, unsigned long long room, unsigned long long& at,
                    unsigned long long& mass) {
    const uint32_t n = ln;
    uint32_t n0 = 0, in = n;      // tokens and mass before the window, tokens in it
    unsigned long long w0 = 0;
    // the window of the order: o in [hi - width, hi]
    unsigned long long hi = by_index ? 0xffffffffull : (unsigned long long)kmax << 32 | 0xffffffffull;
    unsigned long long width = by_index ? (unsigned long long)A.V - 1 : hi - ((unsigned long long)kmin << 32);
    auto order = [&](const Token& t) { return by_index ? t.place & 0xffffffffull : t.place; };
    auto inside = [&](const Token& t) { return t.w != 0 && order(t) <= hi && hi - order(t) <= width; };
    __syncthreads();
    while (in > 64 && width > 0) {
      const int sh = max(0, 64 - __builtin_clzll(width) - 8);
      if (tid < 256) {
        pcount[tid] = 0;
        pmass[tid] = 0;
      }
      __syncthreads();
      for (uint32_t i = tid; i < n; i += NT)
        if (inside(list[i])) {
          const int q = (int)((hi - order(list[i])) >> sh);
          atomicAdd(&pcount[q], 1u);
          atomicAdd(&pmass[q], list[i].w);
        }
      __syncthreads();
      if (wave == 0) {
        uint32_t c[4], cs = 0;
        unsigned long long m[4], ms = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j] = cs += pcount[4 * lane + j];
          m[j] = ms += pmass[4 * lane + j];
        }
        const uint32_t ce = wave_scan(cs), cb = ce - cs, all = lane_value(ce, 63);
        const unsigned long long mb = wave_scan(ms) - ms;
        int best = 255;
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          // (or the last part with a token, where none reaches the mass)
          const bool here = (by_mass ? w0 + mb + m[j] >= room : n0 + cb + c[j] > last) || cb + c[j] == all;
          if (here) best = 4 * lane + j;
          pcount[4 * lane + j] = cb + c[j];
          pmass[4 * lane + j] = mb + m[j];
        }
        best = 255 - (int)wave_max_u(255 - best);
        if (lane == 0) bsh = best;
      }
      __syncthreads();
      const int q = bsh;
      const uint32_t cq = q ? pcount[q - 1] : 0u;
      in = pcount[q] - cq;
      n0 += cq;
      w0 += q ? pmass[q - 1] : 0ull;
      hi -= (unsigned long long)q << sh;
      width = min(width - ((unsigned long long)q << sh), (1ull << sh) - 1);
      __syncthreads();
    }
    // The window's tokens, at most 64 (places are all different), each ranked by 8 lanes
    if (n > 64) {
      if (tid == 0) pcount[0] = 0;
      __syncthreads();
      for (uint32_t i = tid; i < n; i += NT)
        if (inside(list[i])) {
          const uint32_t j = atomicAdd(&pcount[0], 1u);
          if (j < 64) {
            pmass[j] = list[i].place;
            pmass[64 + j] = list[i].w;
          }
        }
      __syncthreads();
    }
    {
      static_assert(NT == 64 * 8, "a token takes 8 lanes");
      const uint32_t np = n > 64 ? min(pcount[0], 64u) : n;
      auto token = [&](uint32_t i) {
        return i >= np ? Token{0, 0} : (n > 64 ? Token{pmass[i], pmass[64 + i]} : list[i]);
      };
      const Token t = token(tid >> 3);
      const unsigned long long mine = order(t);
      uint32_t c = 0;  // the window's kept tokens before this one, and (<< 16) all of them
      unsigned long long m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const Token o = token(8 * j + (tid & 7));
        const bool before = o.w != 0 && order(o) > mine;
        c += (o.w != 0 ? 0x10000u : 0u) + before;
        m += before ? o.w : 0ull;
      }
      c += from_lane<0xb1, 0xf>(c);  // the neighbour's, the neighbour pair's, the other four's (mirrored)
      m += from_lane<0xb1, 0xf>(m);
      c += from_lane<0x4e, 0xf>(c);
      m += from_lane<0x4e, 0xf>(m);
      c += from_lane<0x141, 0xf>(c);
      m += from_lane<0x141, 0xf>(m);
      const uint32_t rank = n0 + (c & 0xffff);
      const bool end = (c & 0xffff) + 1 == c >> 16;  // the window's last
      m += w0;
      const bool cut = by_mass ? (m < room || rank == 0) && (m + t.w >= room || end) : rank == last || (rank < last && end);
      if (t.w != 0 && cut && (tid & 7) == 0) {
        got[0] = t.place;
        got[1] = m + t.w;
      }
    }
    __syncthreads();
    at = got[0];
    mass = got[1];
  };
  auto whole = [](double w) -> unsigned long long { return w > 0.0 ? (unsigned long long)__builtin_ceil(w) : 0ull; };
  // first bin whose tokens take the mass to the goal
  auto bin_at = [&](double goal) -> int {
    __syncthreads();
    if (tid == 0) bsh = NB - 1;
    __syncthreads();
    if (tid < NB && cmass[tid] >= goal && (tid == 0 || cmass[tid - 1] < goal)) bsh = tid;
    __syncthreads();
    return bsh;
  };
  const bool topk = S.k > 0 && (uint32_t)S.k < valid && (uint32_t)S.k <= cum[NB - 2];
  int bk = NB - 1, bm = NB - 1;  // bins of the borders by the histogram
  if (topk) {
    if (tid < NB - 1 && cum[tid] >= (uint32_t)S.k && (tid == 0 || cum[tid - 1] < (uint32_t)S.k)) bsh = tid;
    __syncthreads();
    bk = bsh;
  }
  if (S.m > 0.0) {
    const double d = G.top - floor((double)value_of(mk) * G.s8 + 8.0 * log2(S.m));
    bm = d < (double)(NB - 1) ? max((int)d, 0) : (d != d ? 0 : NB - 1);
  }
  const double least = S.m * weight(G, scale, value_of(mk));  // by min-p
  // Drops what min-p or a place cuts off the list; returns the mass that is left
  auto keep = [&](unsigned long long tp) -> unsigned long long {
    __syncthreads();
    if (tid == 0) fsh = 0;
    __syncthreads();
    unsigned long long w = 0;
    for (uint32_t i = tid; i < ln; i += NT) {
      if (list[i].place < tp || !(weight(G, scale, value_of((uint32_t)(list[i].place >> 32))) >= least)) list[i].w = 0;
      w += list[i].w;
    }
    w = wave_add(w);
    if (lane == 0 && w) atomicAdd(&fsh, w);
    __syncthreads();
    return fsh;
  };

  // Steps: the end of top-k's set, the end of top-p's, and with few candidates, all of them on the list, the draw;
  // else on one border's bin at a time.  (One loop: the selection's code is there once.)
  const bool nucleus = S.p < 1.0 && S.p > 0.0;
  const double enough = S.p * (1.0 - 0x1p-40);  // masses are good to 2^-45 or so: one that meets p exactly has to reach it
  int bc = bk;  // candidates: up to this bin; top-k's border is in the list where top-p's goal needs its set's mass
  if (!(topk && nucleus)) bc = min(min(bk, bm), S.p < 1.0 ? (nucleus ? bin_at(enough * cmass[NB - 1]) : 0) : NB - 1);
  const bool few = bc < NB - 1 && cum[bc] <= CAP;
  int bt = bk;                  // bin of the last token that top-k and top-p keep; NB - 1: none with mass is cut
  unsigned long long tp = 0;    // its place
  double set = cmass[NB - 1];   // mass of top-k's set
  bool ok = true;
  if (S.p <= 0.0) {             // the first token alone
    bt = 0;
    tp = place(mk, mi);
  }
#pragma unroll 1
  for (int step = S.p <= 0.0 || !(topk && (!few || bk == bc)) ? 1 : 0; step < 3 && ok; ++step) {
    unsigned long long q, m, sum = 0, room = 0;
    uint32_t last = 0;
    double above = 0.0;
    int b = bt;
    if (step == 1) {
      if (!nucleus) continue;
      const double goal = enough * set;
      if (!few) {
        b = min(bin_at(goal), bt);
        if (b == NB - 1) continue;
        above = b ? cmass[b - 1] : 0.0;
      }
      room = whole((goal - above) * kFix);
    } else if (step == 0) {
      last = (uint32_t)S.k - 1 - (!few && b ? cum[b - 1] : 0u);
      above = !few && b ? cmass[b - 1] : 0.0;
    } else if (!few) {
      break;
    }
    ok = few ? gather(0, bc) : gather(b, b);
    if (!ok) break;
    if (step == 2) {
      sum = keep(tp);
      room = (unsigned long long)(S.u < 1.0 ? S.u * (double)sum : (double)sum) + 1;
    }
    select(step == 2, step > 0, last, room, q, m);
    if (step == 0) set = above + (double)m * (1.0 / kFix);
    if (step == 2) {
      if (tid == 0) {
        A.ids[r] = (int64_t)(0xffffffffu - (uint32_t)q);
        A.probs[r] = (float)(weight(G, scale, value_of((uint32_t)(q >> 32))) / ((double)sum * (1.0 / kFix)));
      }
      return;
    }
    if (b < bt || q > tp) tp = q;
    bt = b;
  }
  // bins before bf are kept whole, of bf what passes the tests, nothing behind it
  const int bf = min(bt, bm);
  const bool partial = bf < NB - 1;
  if (ok && partial) ok = gather(bf, bf);
  if (!ok) {
    radix_row<T>(A, r, mk, valid, S);
    return;
  }
  auto passes = [&](unsigned long long at, double w) { return at >= tp && w >= least; };
  const double part = partial ? (double)keep(tp) * (1.0 / kFix) : 0.0;
  const double total = (bf > 0 ? cmass[bf - 1] : 0.0) + part;
  const double goal = S.u * total * (1.0 + 0x1p-40);  // a mass that meets it exactly does not pass it

  // the chunk in which the kept mass passes the goal: a wave sums a chunk's whole bins and its listed tokens
  double run = 0.0, start = 0.0, lastrun = 0.0;
  int at = -1, lastc = -1;
  for (int c0 = 0; c0 < nc && at < 0; c0 += NW) {
    if (nc > MC && c0 % MC == 0) shifts(c0);
    const int c = c0 + wave;
    double w = 0.0;
    if (c < nc) {
      const int hi = min(bf - shift[c % MC], NB - 1);
#pragma unroll
      for (int j = 0; j < NB / 64; ++j) {
        const int b = lane + 64 * j;
        w += b < hi ? (double)C[c].mass[b] * scale[b] : 0.0;
      }
      w *= exp2_64(-0.125 * (double)shift[c % MC]);
      if (partial) {
        unsigned long long f = 0;
        for (uint32_t j = lane; j < ln; j += 64)
          if ((0xffffffffu - (uint32_t)list[j].place) / CH == (uint32_t)c) f += list[j].w;
        w += (double)f * (1.0 / kFix);
      }
      w = wave_add(w);
    }
    __syncthreads();
    if (lane == 0) red[wave] = w;
    __syncthreads();
    for (int j = 0; j < NW && c0 + j < nc; ++j) {
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
  // Scan of that chunk: the waves' parts, then the lanes of the part in which the goal is passed, then one lane's tokens
  constexpr int E = CH / NT;
  const int i0 = at * CH + tid * E, i1 = min(A.V, at * CH + CH);
  auto mass_of = [&](int i, float q) -> double {
    const uint32_t k = key_of(q);
    const int b = k != 0 ? G.bin(q) : NB;
    if (!(b < bf || (partial && b == bf))) return 0.0;
    const double w = weight(G, scale, q);
    return b < bf || passes(place(k, i), w) ? w : 0.0;
  };
  double each[E], sum = 0.0;
  {
    T q[E];
    load_tokens<T, E>(x, i0, i1, vec, q);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += each[e] = mass_of(i0 + e, to_f(q[e]));
  }
  const double before = wave_scan(sum) - sum;
  const double all = wave_add(sum);
  __syncthreads();
  if (lane == 0) red[wave] = all;
  __syncthreads();
  int mine = -1;
  double from = 0.0, upto = start;
  for (int j = 0; j < NW; ++j) {
    const double next = upto + red[j];
    if (red[j] > 0.0) {  // (rounding: the last part that has any)
      mine = j;
      from = upto;
      if (next > goal) break;
    }
    upto = next;
  }
  if (wave != mine) return;
  const unsigned long long any = __ballot(sum > 0.0), hit = __ballot(sum > 0.0 && from + before + sum > goal);
  if (lane != (hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any))) return;  // (rounding: the last that has any)
  int found = 0;
  double mass = 0.0, run_ = from + before;
  bool past = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    run_ += each[e];
    if (each[e] > 0.0 && !past) {
      found = i0 + e;
      mass = each[e];
      past = run_ > goal;
    }
  }
  A.ids[r] = found;
  A.probs[r] = (float)(mass / total);
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
  const float* const none = (const float*)ws;  // at least a number for every row
  pa::smp::Args A{x, row, V, u, u64, t ? t : none, k ? k : (const int*)none, p ? p : none, m ? m : none, t0, p0, m0, k0,
                  (t ? 1 : 0) | (k ? 2 : 0) | (p ? 4 : 0) | (m ? 8 : 0), ids, probs};
  const int nc = (V + pa::smp::CH - 1) / pa::smp::CH;
  if (rows * (long long)nc > 0x7fffffff) return (int)hipErrorInvalidValue;
  pa::smp::Chunk* C = (pa::smp::Chunk*)ws;
  PA_DISPATCH_DTYPE(dt, T, {
    pa::smp::chunk_kernel<T><<<(int)(rows * (long long)nc), 256, 0, st>>>(A, C, nc);
    pa::smp::row_kernel<T><<<rows, pa::smp::NT, 0, st>>>(A, C, nc);
  })
  return (int)hipGetLastError();
}
