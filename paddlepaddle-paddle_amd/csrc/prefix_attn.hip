// Attention over a paged KV cache for a batch that shares a prefix: o = softmax([prefix keys, own keys])
// [prefix values, own values], the prefix read once for all sequences.
//
// Mathematics.  A softmax over a union of key sets joins from its parts: with (m, l, a) = (max, sum of
// exp(s - m), sum of exp(s - m) v) of each part, m* = max m, o = sum a exp(m - m*) / sum l exp(m - m*).
// So the work is cut into items, each a tile of query rows against a range of keys:
//   * prefix items: the rows of a key head are ALL its query rows (T tokens x G query heads of the group),
//     cut into tiles of 16 RTP rows; the keys are one range of the shared prefix;
//   * own items: the rows are one sequence's (its n new tokens x G), in tiles of 16 RTO rows; the keys one
//     range of its own pages, up to and including each row's own token (bottom-right causal).
// An item writes (m, l, a) in 32 bits; a second kernel joins a row's items in a fixed order (no atomics).
//
// A block is one item: NW waves, each with a contiguous part of the item's keys and its own stage in LDS,
// so no barrier stands in the key loop.  A wave streams 32-key tiles of K and V by LDS-DMA, the next tile
// in flight while it computes on this one.  S^T = K Q^T on v_mfma_f32_16x16x32 (a lane holds 4 + 4 keys of
// one row: maximum and sum take two lane swaps), P stays in registers as the B operand of O^T = V^T P^T,
// whose A operand is V read transposed (ds_read_b64_tr_b16) in the matching key order.  P is rounded to
// the inputs' type for that product, sums and accumulators are 32-bit.  The base of the exponents lags behind the maximum
// by at most 2^8, and in fp16 lies 2^7 under it: the largest probability is 2^15 at most, and what fp16 drops is 2^-32 of it
// (with a largest of 1 it drops 2^-25, and thousands of keys behind one that takes nearly all are lost).  The NW parts are
// joined in LDS at the end.
//
// Keys past the range and keys of unallocated pages (table entries outside the cache) are read from a row
// of zeros and masked: what lies in a page's unused slots never reaches a product.
//
// Offsets of a block, a head and a slot are 64-bit.  A tile's whole-page path adds its rows' offsets from the first row
// in 32 bits, an instruction's rows in one page likewise; strides for which these do not fit (kTileStride, kRowStride)
// take an address for each lane.
#define PA_FA_PAIR_GROUP_DECL static __constant__
#include "flash_attn_kernels.h"
#include "paged.h"

namespace pa {
namespace pfx {

using fa::f32x4;
using fa::s16x4;
using fa::s16x8;

// Largest slot strides (elements) for which the bytes from a tile's first row to the end of its last one, 63 rows on, are
// under 2^32 (the narrow items' 31 rows: under 2^31), and to the end of a DMA instruction's last row, 7 on, under 2^31
constexpr long long kTileStride = 1ll << 25, kRowStride = 1ll << 27;

__device__ const uint16_t g_zero_row[256] __attribute__((aligned(16))) = {0};

struct Args {
  const uint16_t* q;
  const uint16_t* kc;
  const uint16_t* vc;
  long long qt, qh;            // token / head strides of q
  long long cb, ch, cr;        // block / head / slot strides of both caches
  const int* tables;           // [B, max_blocks]
  long long tstride;
  const int* ptable;           // [pblocks]
  const int* plen_dev;
  const int* lens;
  const int* cu;
  uint16_t* out;               // [T, Hq, D]
  float* lse;                  // [T, Hq] or null
  float* wa;                   // [slots, T Hq, D]
  float2* wml;                 // [slots, T Hq]
  int max_blocks, pblocks, plen, num_blocks, page, page_shift;
  int T, B, Hq, Hkv, G;
  int ntp, nsp, nto, nso;      // row tiles and key ranges of the two kinds
  int most;                    // new tokens of a sequence at most
  float scale;                 // log2 units
};

// Keys per range when `len` keys are cut into at most n ranges: a multiple of 32 keys a wave, and no range
// shorter than two tiles a wave (a shorter one costs more to join than to read).
__host__ __device__ __forceinline__ int range_keys(int len, int n, int nw) {
  const int per = (int)(((long long)len + n - 1) / n), unit = 32 * nw;
  const int r = (per + unit - 1) / unit * unit;
  return r < 2 * unit ? 2 * unit : r;
}

__device__ __forceinline__ int prefix_len(const Args& A) {
  const long long cap = (long long)A.pblocks * A.page;
  const int p = A.plen_dev ? *A.plen_dev : A.plen;
  return p < 0 ? 0 : (int)min((long long)p, cap);
}
__device__ __forceinline__ int own_len(const Args& A, int b) {
  const long long cap = (long long)A.max_blocks * A.page;
  const int p = A.lens[b];
  return p < 0 ? 0 : (int)min((long long)p, cap);
}

// One 16-B-per-lane LDS-DMA from a per-lane 64-bit address (fa_glds takes a base that all lanes share)
__device__ __forceinline__ void glds64(const void* src, unsigned lds_dst) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(src), "s"(lds_dst)
      : "memory");
}

template <typename T>
constexpr float kUp = __is_same(T, f16_t) ? 7.f : 0.f;  // log2 of a probability whose score is the base's maximum

// Weight of a part (m, l) in a join to maximum M.  A part that saw no key has m = -inf and l = 0; one whose
// scores were all NaN has m = -inf and l = NaN, which has to reach the result.
__device__ __forceinline__ float part_weight(float2 ml, float M) {
  return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : NAN) : fa::fast_exp2(ml.x - M);
}
// 1 / l; 0 for a row that saw no key; NaN stays NaN
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : NAN); }
__device__ __forceinline__ float row_lse(float M, float l) {
  return l > 0.f ? (M + __builtin_amdgcn_logf(l)) * fa::kLn2 : (l == 0.f ? -INFINITY : NAN);
}

// The N DMA instructions of a tile whose rows lie in one page: instruction i writes 1 KiB at dst + 1024 i from
// base + off[i] + 1024 (i % 4).  The instruction's own offset moves both ends, so M0 changes every fourth time.
template <int N>
__device__ __forceinline__ void dma_tile(const char* base, const unsigned (&off)[N], unsigned dst) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %5\n\t"
        "global_load_lds_dwordx4 %2, %5 offset:1024\n\t"
        "global_load_lds_dwordx4 %3, %5 offset:2048\n\t"
        "global_load_lds_dwordx4 %4, %5 offset:%7\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(off[i]), "v"(off[i + 1]), "v"(off[i + 2]), "v"(off[i + 3]), "s"(base), "s"(dst + i * 1024),
          "n"(3 * 1024)
        : "memory");
  }
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// maximum over the four lane groups g = lane >> 4 of a column
__device__ __forceinline__ float groups_max(float v) {
  // lane swaps instead of two trips through LDS; s_nop: a VALU result is read by a lane swap
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  a = b = fmaxf(a, b);
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}

// Operands from the LDS images of K and V tiles, by 32-bit LDS addresses.  A lane's address in the swizzled image is
// one constant, with the operand's number put over it by an exclusive or (the images are those of fa::lds_off).
typedef __attribute__((address_space(3))) const char lds_char;
template <int D>
__device__ __forceinline__ unsigned row_base(int lane) {  // K: row lane & 15, 8 values from 8 (lane >> 4) on
  const int r = lane & 15, sw = fa::swz_b128<D>(r);
  return (unsigned)(r * D * 2 + ((((lane >> 4) ^ sw) & 3) << 4) + ((sw >> 2) << 6));
}
template <int D>
__device__ __forceinline__ s16x8 read_row(unsigned tile, unsigned base, int h, int k) {  // rows 16 h .., values 32 k ..
  return *(__attribute__((address_space(3))) const s16x8*)(tile + (base ^ (unsigned)(k << 6)) + (unsigned)(h * 16 * D * 2));
}
template <int D>
__device__ __forceinline__ unsigned col_base(int lane) {  // V transposed: row 4 (lane >> 4) + lane / 4 % 4, columns 4 (lane % 4) ..
  const int r = 4 * (lane >> 4) + ((lane >> 2) & 3), p = lane & 3;
  return (unsigned)(r * D * 2 + (p >> 1) * 16 + (p & 1) * 8 + (fa::swz_tr<D>(r) << 4));
}
template <int D>
__device__ __forceinline__ s16x8 read_col(unsigned tile, unsigned base, int j, int d) {  // rows 32 j .., columns 16 d ..
  typedef __attribute__((address_space(3))) s16x4 lds_v4;
  const unsigned at = tile + (base ^ (unsigned)(d << 5)) + (unsigned)(32 * j * D * 2);
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)at);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(at + 16 * D * 2));
  return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Pages of a wave's key range: 64 table entries in a register, one per lane
struct Window {
  const int* table;
  int count, w0, val;
  __device__ __forceinline__ void load(int p) {
    w0 = p;
    const int i = p + (int)(threadIdx.x & 63);
    val = i < count ? table[i] : -1;
    // waited for here, where it is rare: at its uses the compiler's wait would drain the tiles in flight too
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(val)::"memory");
  }
  __device__ __forceinline__ int at(int p) const { return __shfl(val, p - w0, 64); }
};

template <typename T, int D, int NW>
struct Shared {
  static constexpr int TILE = 32 * D * 2;       // bytes of 32 keys
  static constexpr int STAGE = 2 * TILE;        // K and V
  static constexpr int RPI = 1024 / (D * 2);    // rows of one DMA instruction
  static constexpr int NI = 32 / RPI;           // DMA instructions of a tile
  static constexpr int OP = D + 4;              // row pitch of the joined accumulators (floats)
};
template <int RT, int D, int NW>
constexpr int lds_bytes() {
  constexpr int stage = NW * 2 * 32 * D * 2, join = NW * 16 * (D + 4) * 4;
  return (stage > join ? stage : join) + NW * RT * 16 * 8 + RT * 16 * D;
}

// What bounds it: the read of its keys and values where rows are few (own pages of 256 sequences of 500 .. 1500 keys,
// 8 heads of 128: 218 us, 4.85 TB/s); the launch and three dependent loads for a small call (4 sequences of 32 heads
// behind 1000 keys: 10 us, and 4 for the join).
// One item: rows [row0, row0 + 16 RT) of `nrows` rows (row r = token tok0 + r / G, head hk G + r % G)
// against keys [k0, k1) of `table`; row r sees keys < lim0 + r / G (CAUSAL) or all.
template <typename T, int D, int RT, int NW, bool CAUSAL>
__device__ __forceinline__ void item(const Args& A, char* smem, int hk, int tok0, int row0, int nrows, int k0, int k1,
                                     const int* table, int tcount, int lim0, int slot, bool direct) {
  using SH = Shared<T, D, NW>;
  constexpr int KS = D / 32, DB = D / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;

  // queries: B operand of S^T, lane holds Q[row c16][32 ks + 8 g .. + 8]
  s16x8 qf[RT][KS];
  int lim[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = row0 + 16 * t + c16, i = r / A.G;
    lim[t] = r < nrows ? (CAUSAL ? lim0 + i : k1) : 0;
    const uint16_t* p = A.q + (long long)(tok0 + i) * A.qt + (long long)(hk * A.G + r % A.G) * A.qh + 8 * g;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      qf[t][k] = r < nrows ? *reinterpret_cast<const s16x8*>(p + 32 * k) : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
  // the first key that some row of the tile does not see
  const int full = CAUSAL ? lim0 + row0 / A.G : k1;

  f32x4 acc[RT][DB];            // O^T
  float l[RT];                  // sum of this lane's probabilities, before they are rounded
  float nm[RT], thr[RT];        // minus the base of the exponents (the maximum - kUp); the score at which it has to move
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    nm[t] = 0.f;
    thr[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // LDS: the waves' stages, later the parts to be joined; (m, l) of each wave and row; what of a row's values
  // was not finite (bits 0, 1, 2 of a byte: +inf, -inf, NaN)
  float2* const ml = reinterpret_cast<float2*>(smem + lds_bytes<RT, D, NW>() - NW * RT * 16 * 8 - RT * 16 * D);
  unsigned* const notes = reinterpret_cast<unsigned*>(smem + lds_bytes<RT, D, NW>() - RT * 16 * D);
  if constexpr (CAUSAL) {
    for (int i = threadIdx.x; i < RT * 16 * D / 4; i += NW * 64) notes[i] = 0;
    __syncthreads();
  }

  // this wave's keys
  const int per = ((k1 - k0 + NW - 1) / NW + 31) / 32 * 32;
  const int ka = min(k0 + wave * per, k1), kb = min(ka + per, k1);
  const int nt = (kb - ka + 31) / 32;
  char* const st = smem + wave * SH::STAGE;  // K, V
  const unsigned st32 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)st);
  const int rl = lane / (D / 8), cl = lane % (D / 8);  // row of a DMA instruction, chunk that this lane writes
  const char* const kh = reinterpret_cast<const char*>(A.kc + hk * A.ch);
  const char* const vh = reinterpret_cast<const char*>(A.vc + hk * A.ch);
  auto page_of = [&](int key) { return A.page_shift >= 0 ? key >> A.page_shift : key / A.page; };

  Window win{table, tcount, 0, -1};
  if (nt > 0) win.load(page_of(ka));

  // LDS-DMA of the 32 keys (or values) from kt on into the LDS image at dst: NI instructions on every path.
  // A lane fetches chunk cl ^ swizzle of its row; the swizzle is that of the image.  Returns the keys (bit r:
  // key kt + r) that exist.
  const bool whole_page = A.page % 32 == 0 && A.cr >= D && A.cr <= kTileStride,
             grouped = A.page % SH::RPI == 0 && A.cr <= kRowStride;
  unsigned fk[SH::NI], fv[SH::NI];  // byte offsets of the fast path, less what the instruction's offset adds
#pragma unroll
  for (int i = 0; i < SH::NI; ++i) {
    const int row = i * SH::RPI + rl;
    const unsigned r = (unsigned)row * (unsigned)A.cr * 2 - (i & 3) * 1024;
    fk[i] = r + ((unsigned)(cl ^ fa::swz_b128<D>(row)) << 4);
    fv[i] = r + ((unsigned)(cl ^ fa::swz_tr<D>(row)) << 4);
  }
  auto slow = [&](auto isv, int kt, unsigned dst) -> unsigned {
    const char* const base = isv ? vh : kh;
    const int p1 = page_of(min(kt + 31, kb - 1));
    if (p1 - win.w0 >= 64) win.load(page_of(kt));
    const int key = kt + (lane & 31), pg = min(page_of(key), p1), blk = win.at(pg);
    const unsigned ok = (unsigned)__ballot(key < kb && (unsigned)blk < (unsigned)A.num_blocks);
    const unsigned long long off = (unsigned long long)((long long)blk * A.cb + (long long)(key - pg * A.page) * A.cr) * 2;
    const unsigned lo = (unsigned)off, hi = (unsigned)(off >> 32);
    if (ok == 0xffffffffu && grouped) {  // the rows of an instruction lie in one page: a scalar base for each
#pragma unroll
      for (int i = 0; i < SH::NI; ++i) {
        // (unsigned): readlane gives an int, whose sign would reach the upper half
        const unsigned long long o = (unsigned long long)(unsigned)__builtin_amdgcn_readlane(lo, i * SH::RPI) |
                                     (unsigned long long)(unsigned)__builtin_amdgcn_readlane(hi, i * SH::RPI) << 32;
        const int row = i * SH::RPI + rl;
        const unsigned sw = (unsigned)(cl ^ (isv ? fa::swz_tr<D>(row) : fa::swz_b128<D>(row))) << 4;
        fa::fa_glds(base + o, (unsigned)rl * (unsigned)A.cr * 2 + sw, dst + i * 1024);
      }
    } else {  // an address for each lane; rows that do not exist come from a row of zeros
      int ln = lane;
      asm volatile("" : "+v"(ln));  // rare: its addresses are formed here, not kept in registers through the loop
#pragma unroll
      for (int i = 0; i < SH::NI; ++i) {
        const int row = i * SH::RPI + ln / (D / 8);
        const unsigned long long o = (unsigned long long)(unsigned)__shfl((int)lo, row, 64) |
                                     (unsigned long long)(unsigned)__shfl((int)hi, row, 64) << 32;
        const unsigned sw = (unsigned)((ln % (D / 8)) ^ (isv ? fa::swz_tr<D>(row) : fa::swz_b128<D>(row))) << 4;
        glds64(((ok >> row) & 1) ? base + o + sw : reinterpret_cast<const char*>(g_zero_row) + sw, dst + i * 1024);
      }
    }
    return ok;
  };
  auto issue = [&](auto isv, int kt, unsigned dst) -> unsigned {
    if (whole_page && kt + 32 <= kb) {  // 32 keys of one page
      const int p = page_of(kt);
      if (p - win.w0 >= 64) win.load(p);
      const unsigned blk = __builtin_amdgcn_readlane(win.val, p - win.w0);
      if (blk < (unsigned)A.num_blocks) {
        const char* base = (isv ? vh : kh) + ((long long)blk * A.cb + (long long)(kt - p * A.page) * A.cr) * 2;
        dma_tile<SH::NI>(base, isv ? fv : fk, dst);
        return 0xffffffffu;
      }
    }
    return slow(isv, kt, dst);
  };
  std::false_type isk;
  std::true_type isv;

  const unsigned dk = st32, dv = st32 + SH::TILE;
  const char* const vbuf = st + SH::TILE;
  const unsigned rb = row_base<D>(lane), cb = col_base<D>(lane);
  unsigned ok = 0;
  if (nt > 0) {
    ok = issue(isk, ka, dk);
    issue(isv, ka, dv);
  }
  for (int it = 0; it < nt; ++it) {
    const int kt = ka + 32 * it;
    const unsigned here = ok;
    const bool more = it + 1 < nt;
    wait_vm<SH::NI>();  // K is here; V may be on its way
    f32x4 s[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const s16x8 a0 = read_row<D>(dk, rb, 0, k), a1 = read_row<D>(dk, rb, 1, k);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        s[t][0] = fa::Mfma<T>::run(a0, qf[t][k], s[t][0]);
        s[t][1] = fa::Mfma<T>::run(a1, qf[t][k], s[t][1]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read: the next may come
    if (more) ok = issue(isk, kt + 32, dk);
    if (here != 0xffffffffu || kt + 32 > full) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 16 * h + 4 * g + e;
            if (!((here >> (4 * g)) & (1u << (16 * h + e))) || kt + r >= lim[t]) s[t][h][e] = -INFINITY;
          }
    }
    // The base moves only when a score outgrows it by 2^8; whether one does needs no look at other lanes.
    float over = -INFINITY, mx[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      // v_maximum3_f32 (a NaN stays: such a row ends as NaN whatever its base is)
      mx[t] = max3(max3(max3(s[t][0][0], s[t][0][1], s[t][0][2]), s[t][0][3], s[t][1][0]),
                   max3(s[t][1][1], s[t][1][2], s[t][1][3]), -INFINITY);
      over = fmaxf(over, mx[t] * A.scale - thr[t]);  // NaN (nothing seen, nothing here) is passed over
    }
    if (__ballot(over > 0.f)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float m1 = groups_max(mx[t]) * A.scale;
        const bool mv = m1 > thr[t];
        const float f = thr[t] == -INFINITY ? 0.f : (mv ? fa::fast_exp2(kUp<T> - nm[t] - m1) : 1.f);
        if (mv) {
          nm[t] = kUp<T> - m1;
          thr[t] = m1 + fa::kRescaleTau;
        }
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[t][d] *= f;
      }
    }
    s16x8 pf[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float p[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[h][e] = fa::fast_exp2(s[t][h][e] * A.scale + nm[t]);
      l[t] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
      unsigned w[4];
      w[0] = fa::f2s2<T>(p[0][0], p[0][1]);
      w[1] = fa::f2s2<T>(p[0][2], p[0][3]);
      w[2] = fa::f2s2<T>(p[1][0], p[1][1]);
      w[3] = fa::f2s2<T>(p[1][2], p[1][3]);
      pf[t] = __builtin_bit_cast(s16x8, w);
    }
    if (more) wait_vm<SH::NI>();  // V is here; the next K may be on its way
    else wait_vm<0>();
    bool odd = false;
    if constexpr (CAUSAL) {
      // a tile that some rows see in part: its values may hold an infinity or a NaN of a later token, which
      // a zero probability in a product would carry into the earlier tokens' rows
      if (kt + 32 > full) {
        constexpr unsigned EX = __is_same(T, f16_t) ? 0x7c00u : 0x7f80u;
        for (int i = lane; i < SH::TILE / 16; i += 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(vbuf + i * 16);
          const unsigned w4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) odd |= (w4[j] & EX) == EX || ((w4[j] >> 16) & EX) == EX;
        }
      }
      odd = __ballot(odd) != 0;
      if (odd) {
        // which rows meet an infinity or a NaN: products with 1 in their places and 0 elsewhere, noted in LDS
        // and brought into the row at the join; the product below then takes the finite values alone
        constexpr short ONE = __is_same(T, f16_t) ? 0x3c00 : 0x3f80, INF = __is_same(T, f16_t) ? 0x7c00 : 0x7f80;
#pragma unroll 1
        for (int d = 0; d < DB; ++d) {
          const s16x8 v = read_col<D>(dv, cb, 0, d);
          unsigned note[RT];
#pragma unroll
          for (int t = 0; t < RT; ++t) note[t] = 0;
#pragma unroll
          for (int kind = 0; kind < 3; ++kind) {
            s16x8 x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const bool inf = (v[j] & 0x7fff) == INF, nan = (v[j] & 0x7fff) > INF;
              x[j] = (kind == 0 ? inf && v[j] > 0 : (kind == 1 ? inf && v[j] < 0 : nan)) ? ONE : (short)0;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              const f32x4 z = fa::Mfma<T>::run(x, pf[t], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int e = 0; e < 4; ++e) note[t] |= z[e] > 0.f ? 1u << (8 * e + kind) : 0u;
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) atomicOr(&notes[(16 * t + c16) * (D / 4) + 4 * d + g], note[t]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int i = lane; i < SH::TILE / 4; i += 64) {
          unsigned* const w = reinterpret_cast<unsigned*>(const_cast<char*>(vbuf)) + i;
          const unsigned x = *w;
          *w = ((x & 0x7fffu) >= (unsigned)INF ? 0u : x & 0xffffu) |
               (((x >> 16) & 0x7fffu) >= (unsigned)INF ? 0u : x & 0xffff0000u);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const s16x8 v = read_col<D>(dv, cb, 0, d);
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t][d] = fa::Mfma<T>::run(v, pf[t], acc[t][d]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
    if (more) issue(isv, kt + 32, dv);
  }
  float m[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) m[t] = thr[t] == -INFINITY ? -INFINITY : -nm[t];

  // join the waves' parts
  float* const oj = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);  // over the lane groups
    l[t] += __shfl_xor(l[t], 32, 64);
    if (g == 0) ml[(wave * RT + t) * 16 + c16] = make_float2(m[t], l[t]);
  }
  __syncthreads();  // every wave is past its stage
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (t > 0) __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[(w * RT + t) * 16 + c16].x);
    const float f = part_weight(make_float2(m[t], l[t]), M);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *reinterpret_cast<f32x4*>(oj + (wave * 16 + c16) * SH::OP + 16 * d + 4 * g) = acc[t][d] * f;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += NW * 64) {
      const int rr = i / (D / 4), d = (i % (D / 4)) * 4, r = row0 + 16 * t + rr;
      if (r >= nrows) continue;
      float Mr = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) Mr = fmaxf(Mr, ml[(w * RT + t) * 16 + rr].x);
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 x = ml[(w * RT + t) * 16 + rr];
        L += x.y * part_weight(x, Mr);
        o += *reinterpret_cast<const f32x4*>(oj + (w * 16 + rr) * SH::OP + d);
      }
      if constexpr (CAUSAL) {
        const unsigned n = notes[(16 * t + rr) * (D / 4) + d / 4];
        if (n != 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (n >> (8 * e) & 1) o[e] += INFINITY;
            if (n >> (8 * e) & 2) o[e] -= INFINITY;
            if (n >> (8 * e) & 4) o[e] = NAN;
          }
      }
      const long long row = (long long)(tok0 + r / A.G) * A.Hq + hk * A.G + r % A.G;
      if (direct) {
        const float k = inverse_sum(L);
        if (L == 0.f) o = f32x4{0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<uint2*>(A.out + row * D + d) =
            make_uint2(fa::f2s2<T>(o[0] * k, o[1] * k), fa::f2s2<T>(o[2] * k, o[3] * k));
        if (A.lse && d == 0) A.lse[row] = row_lse(Mr, L);
      } else {
        *reinterpret_cast<f32x4*>(A.wa + ((long long)slot * A.T * A.Hq + row) * D + d) = o;
        if (d == 0) A.wml[(long long)slot * A.T * A.Hq + row] = make_float2(Mr, L);
      }
    }
  }
}

// A prefix item of many rows: the NW waves share each tile of 64 keys, two of which are in LDS, and have 16 RT
// rows of their own: rows [row0, row0 + 16 RT NW) against keys [k0, k1), all of which every row sees.  In the
// layout of item() each wave reads all of its own keys from L2, 32 rows at a time: at 2048 rows a key head that
// is 19 TB/s of L2 reads, which bound it (518 TFLOP/s); here a tile serves 8 times as many rows (860 TFLOP/s for 256
// queries of 64 heads behind 32768 keys of 8 heads, 128 values each).  What bounds it now: no one thing; without the
// DMA, the barrier, the exponentials, the value product or the LDS reads alone it takes 84 to 94 % of its time, and 256
// registers leave two waves a SIMD to cover each other's waits.
constexpr int kWideRT = 2;
// Tiles between two meetings of a block's waves: what LDS holds in rings of twice as many
template <int D>
constexpr int wide_depth() {
  return D <= 64 ? 2 : 1;
}

// Asks the scheduler for N times one matrix instruction, three vector ones and an exponential behind it: the
// matrix cores run while the wave issues the others
template <int N>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
    __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
  }
}

template <typename T, int D, int RT, int NW>
__device__ __forceinline__ void wide_item(const Args& A, char* smem, int hk, int row0, int nrows, int k0, int k1, int slot) {
  using SH = Shared<T, D, NW>;
  constexpr int KS = D / 32, DB = D / 16, TILE = 64 * D * 2, ND = 64 / SH::RPI / NW;  // DMA instructions a wave, K or V
  static_assert(ND * SH::RPI * NW == 64, "a tile's rows divide over the waves");
  constexpr int DEPTH = wide_depth<D>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  row0 += wave * 16 * RT;
  s16x8 qf[RT][KS];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = row0 + 16 * t + c16;
    const uint16_t* p = A.q + (long long)(r / A.G) * A.qt + (long long)(hk * A.G + r % A.G) * A.qh + 8 * g;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      qf[t][k] = r < nrows ? *reinterpret_cast<const s16x8*>(p + 32 * k) : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
  f32x4 acc[RT][DB];
  float l[RT], nm[RT], thr[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    nm[t] = l[t] = 0.f;
    thr[t] = -INFINITY;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int nt = (k1 - k0 + 63) / 64;
  const unsigned st32 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)smem);
  const int rl = lane / (D / 8), cl = lane % (D / 8);
  const char* const kh = reinterpret_cast<const char*>(A.kc + hk * A.ch);
  const char* const vh = reinterpret_cast<const char*>(A.vc + hk * A.ch);
  auto page_of = [&](int key) { return A.page_shift >= 0 ? key >> A.page_shift : key / A.page; };
  const bool grouped = A.page % SH::RPI == 0 && A.cr <= kRowStride;
  Window win{A.ptable, A.pblocks, 0, -1};
  if (nt > 0) win.load(page_of(k0));
  unsigned sk[ND], sv[ND];  // byte offsets from the first row of an instruction
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int row = (wave * ND + i) * SH::RPI + rl;
    sk[i] = (unsigned)rl * (unsigned)A.cr * 2 + ((unsigned)(cl ^ fa::swz_b128<D>(row)) << 4);
    sv[i] = (unsigned)rl * (unsigned)A.cr * 2 + ((unsigned)(cl ^ fa::swz_tr<D>(row)) << 4);
  }

  // Places of a tile's 64 keys: byte offset of key kt + lane from the head's base, and which keys exist
  struct Places {
    unsigned lo, hi;
    unsigned long long ok;
  };
  const bool aligned = A.page % 64 == 0 && A.cr <= kTileStride;  // a tile lies in one page
  const unsigned lane_off = (unsigned)lane * (unsigned)A.cr * 2;
  auto places = [&](int kt) -> Places {
    if (aligned) {
      const int p = page_of(kt);
      if (p - win.w0 >= 64) win.load(p);
      const int blk = __builtin_amdgcn_readlane(win.val, p - win.w0);
      const unsigned long long off =
          (unsigned long long)((long long)blk * A.cb + (long long)(kt - p * A.page) * A.cr) * 2 + lane_off;
      return Places{(unsigned)off, (unsigned)(off >> 32),
                    (unsigned)blk < (unsigned)A.num_blocks ? (unsigned long long)__ballot(kt + lane < k1) : 0ull};
    }
    const int p1 = page_of(min(kt + 63, k1 - 1));
    if (p1 - win.w0 >= 64) win.load(page_of(kt));  // 64 pages hold a tile
    const int key = kt + lane, pg = min(page_of(key), p1), blk = win.at(pg);
    const unsigned long long off = (unsigned long long)((long long)blk * A.cb + (long long)(key - pg * A.page) * A.cr) * 2;
    return Places{(unsigned)off, (unsigned)(off >> 32),
                  (unsigned long long)__ballot(key < k1 && (unsigned)blk < (unsigned)A.num_blocks)};
  };
  // this wave's rows of a tile's K (or V)
  auto issue = [&](auto isv, const Places& p, unsigned dst) {
    const char* const base = isv ? vh : kh;
    dst += wave * ND * 1024;
    if (p.ok == ~0ull && grouped) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int r = (wave * ND + i) * SH::RPI;
        const unsigned long long o = (unsigned long long)(unsigned)__builtin_amdgcn_readlane(p.lo, r) |
                                     (unsigned long long)(unsigned)__builtin_amdgcn_readlane(p.hi, r) << 32;
        fa::fa_glds(base + o, isv ? sv[i] : sk[i], dst + i * 1024);
      }
    } else {
      int ln = lane;
      asm volatile("" : "+v"(ln));  // rare: its addresses are formed here, not kept in registers through the loop
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int r = (wave * ND + i) * SH::RPI + ln / (D / 8);
        const unsigned sw = (unsigned)((ln % (D / 8)) ^ (isv ? fa::swz_tr<D>(r) : fa::swz_b128<D>(r))) << 4;
        const unsigned long long o = (unsigned long long)(unsigned)__shfl((int)p.lo, r, 64) |
                                     (unsigned long long)(unsigned)__shfl((int)p.hi, r, 64) << 32;
        glds64(((p.ok >> r) & 1) ? base + o + sw : reinterpret_cast<const char*>(g_zero_row) + sw, dst + i * 1024);
      }
    }
  };

  std::false_type isk;
  std::true_type isv;
  f32x4 s[RT][4], c[RT][4];
  float mx[RT], over = -INFINITY;
  const unsigned rb = row_base<D>(lane), cb = col_base<D>(lane);
  auto scores = [&](unsigned kbuf, f32x4 (&o)[RT][4]) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 4; ++h) o[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const s16x8 a = read_row<D>(kbuf, rb, h, k);
#pragma unroll
        for (int t = 0; t < RT; ++t) o[t][h] = fa::Mfma<T>::run(a, qf[t][k], o[t][h]);
      }
  };
  auto mask = [&](unsigned long long ok, f32x4 (&o)[RT][4]) {
    if (ok != ~0ull) {
      const unsigned long long mine = ok >> (4 * g);  // key 16 h + 4 g + e at bit 16 h + e
      const unsigned w[2] = {(unsigned)mine, (unsigned)(mine >> 32)};
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(w[h >> 1] & (1u << (16 * (h & 1) + e)))) o[t][h][e] = -INFINITY;
    }
  };
  auto maxima = [&](const f32x4 (&o)[RT][4]) {
    over = -INFINITY;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float a = max3(max3(o[t][0][0], o[t][0][1], o[t][0][2]), o[t][0][3], o[t][1][0]);
      const float b = max3(max3(o[t][1][1], o[t][1][2], o[t][1][3]), o[t][2][0], o[t][2][1]);
      const float d = max3(max3(o[t][2][2], o[t][2][3], o[t][3][0]), o[t][3][1], o[t][3][2]);
      mx[t] = max3(max3(a, b, d), o[t][3][3], o[t][3][3]);
      over = fmaxf(over, mx[t] * A.scale - thr[t]);
    }
  };
  auto rebase = [&] {
    if (__ballot(over > 0.f)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float m1 = groups_max(mx[t]) * A.scale;
        const bool mv = m1 > thr[t];
        const float f = thr[t] == -INFINITY ? 0.f : (mv ? fa::fast_exp2(kUp<T> - nm[t] - m1) : 1.f);
        if (mv) {
          nm[t] = kUp<T> - m1;
          thr[t] = m1 + fa::kRescaleTau;
        }
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[t][d] *= f;
      }
    }
  };

  // LDS: rings of 2 DEPTH tiles of K and of V.  Pipeline: while a tile's probabilities are formed, the next tile's
  // scores are on the matrix cores.  The waves meet once in DEPTH tiles, and fetch as many.
  constexpr int RING = 2 * DEPTH;
  const unsigned kr = st32, vr = st32 + RING * TILE;
  auto exists = [&](int t) { return t < nt; };
  auto tile = [&](int it, auto u, const f32x4 (&s)[RT][4], f32x4 (&c)[RT][4], unsigned long long ok) {
    const unsigned kbuf = kr + ((DEPTH == 1 ? u + 1 : it + 1) % RING) * TILE;
    const unsigned vbuf = vr + ((DEPTH == 1 ? u : it) % RING) * TILE;
    // Phase 1: FG RT products a step with a part of the probabilities under them, the operands of the next step on
    // their way from LDS; phase 2: the product with the values, likewise a step ahead.  The barriers keep
    // the compiler from sinking each read to its product, where a wave would wait out the LDS's latency 48
    // times a tile.  (Behind the last tile the scores are of stale bytes, and never used.)
    constexpr int FG = D == 256 ? 4 : 2, NK = 4 * KS / FG, NV = 2 * DB / FG;  // operands a step, steps of the phases
    s16x8 pf[RT][2], fr[2][FG];
    auto read = [&](int step, s16x8 (&f)[FG]) {  // operand i of phase 1: keys 16 (i % 4), values 32 (i / 4) of K
#pragma unroll
      for (int j = 0; j < FG; ++j) {
        const int i = step * FG + j, v = i - 4 * KS;
        f[j] = v < 0 ? read_row<D>(kbuf, rb, i & 3, i >> 2) : read_col<D>(vbuf, cb, v / DB, v % DB);
      }
    };
    read(0, fr[0]);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 4; ++h) c[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      read(k + 1, fr[(k + 1) & 1]);
#pragma unroll
      for (int j = 0; j < FG; ++j) {
        const int i = k * FG + j;
#pragma unroll
        for (int t = 0; t < RT; ++t) c[t][i & 3] = fa::Mfma<T>::run(fr[k & 1][j], qf[t][i >> 2], c[t][i & 3]);
      }
#pragma unroll
      for (int i = 0; i < 4 * RT; ++i)  // part i of the probabilities: row tile i / 4, 16 keys i % 4
        if (i * NK / (4 * RT) == k) {
          const int t = i / 4, h = i % 4;
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = fa::fast_exp2(s[t][h][e] * A.scale + nm[t]);
          l[t] += (p[0] + p[1]) + (p[2] + p[3]);
          const unsigned w[2] = {fa::f2s2<T>(p[0], p[1]), fa::f2s2<T>(p[2], p[3])};
          const s16x4 q = __builtin_bit_cast(s16x4, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) pf[t][h / 2][4 * (h % 2) + e] = q[e];
        }
      interleave<FG * RT>();
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (q + 1 < NV) read(NK + q + 1, fr[(NK + q + 1) & 1]);
#pragma unroll
      for (int j = 0; j < FG; ++j) {
        const int i = q * FG + j;  // values 16 (i % DB) of keys 32 (i / DB)
#pragma unroll
        for (int t = 0; t < RT; ++t)
          acc[t][i % DB] = fa::Mfma<T>::run(fr[(NK + q) & 1][j], pf[t][i / DB], acc[t][i % DB]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (exists(it + 1)) {
      mask(ok, c);
      maxima(c);
      rebase();
    }
  };
  Places ahead{0, 0, 0};         // of the last tile whose K was asked for
  unsigned long long ok1 = 0, next = 0;  // keys of the next tile (DEPTH 2), and of the one after the next two
  if (nt > 0) {
    Places pl = places(k0);
    const unsigned long long ok0 = pl.ok;
    issue(isk, pl, kr);
    issue(isv, pl, vr);
#pragma unroll
    for (int t = 1; t <= DEPTH; ++t)
      if (exists(t)) {
        ahead = places(k0 + 64 * t);
        if (t == 1) ok1 = ahead.ok;
        issue(isk, ahead, kr + t * TILE);
        if (t < DEPTH) issue(isv, ahead, vr + t * TILE);
      }
    wait_vm<0>();
    __syncthreads();
    scores(kr, s);
    mask(ok0, s);
    maxima(s);
    rebase();
  }
  for (int it = 0; it < nt; it += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = it + u;
      if (!exists(i)) break;
      unsigned long long m = ok1;  // keys of tile i + 1
      if (u % DEPTH == 0) {
        wait_vm<0>();
        __syncthreads();  // what was asked for is here, and every wave is done with what it replaces
        if constexpr (DEPTH == 1) m = ahead.ok;
        if (exists(i + DEPTH)) issue(isv, ahead, vr + (i + DEPTH) % RING * TILE);
        if constexpr (DEPTH == 2) ok1 = ahead.ok;
        if (exists(i + DEPTH + 1)) {
          ahead = places(k0 + 64 * (i + DEPTH + 1));
          issue(isk, ahead, kr + (i + DEPTH + 1) % RING * TILE);
          if constexpr (DEPTH == 2) {
            issue(isv, ahead, vr + (i + 3) % RING * TILE);
            next = ahead.ok;
            if (exists(i + 4)) {
              ahead = places(k0 + 64 * (i + 4));
              issue(isk, ahead, kr + (i + 4) % RING * TILE);
            }
          }
        }
      } else {
        ok1 = next;
      }
      if (u == 0) tile(i, std::integral_constant<int, 0>{}, s, c, m);
      else tile(i, std::integral_constant<int, 1>{}, c, s, m);
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    const int r = row0 + 16 * t + c16;
    if (r >= nrows) continue;
    const long long row = (long long)slot * A.T * A.Hq + (long long)(r / A.G) * A.Hq + hk * A.G + r % A.G;
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(A.wa + row * D + 16 * d + 4 * g) = acc[t][d];
    if (g == 0) A.wml[row] = make_float2(thr[t] == -INFINITY ? -INFINITY : -nm[t], l[t]);
  }
}

__device__ __forceinline__ void seq_rows(const Args& A, int b, int& tok0, int& n) {
  tok0 = A.cu ? A.cu[b] : b;
  n = A.cu ? A.cu[b + 1] - tok0 : 1;
  if (tok0 < 0 || tok0 > A.T || n < 0 || n > A.most || tok0 + n > A.T) n = 0;  // offsets that do not fit the call: nothing is read
}

// Items in the order of dispatch, 8 blocks at a time (one per XCD): the prefix items, which take longest, then the
// own ones.  (Blocks go to the shader engines of an XCD in turn: an alternation of the kinds puts all the long ones
// on some of them, and the others wait.)  Each XCD has a contiguous part of the items, whose row tiles over the same
// keys are neighbours and meet in its L2.
// RTP = 0: wide prefix items (of kWideRT row tiles a wave)
template <typename T, int D, int RTP, int RTO, int NW>
__global__ __launch_bounds__(NW * 64) void items_kernel(Args A) {
  constexpr int RTM = RTP > RTO ? RTP : RTO, narrow = lds_bytes<RTM, D, NW>(), wide = RTP == 0 ? 4 * wide_depth<D>() * 64 * D * 2 : 0;
  __shared__ __attribute__((aligned(16))) char smem[narrow > wide ? narrow : wide];
  const int np = A.Hkv * A.ntp * A.nsp, no = A.B * A.Hkv * A.nto * A.nso;
  const int gp = (np + 7) / 8, go = (no + 7) / 8, x = blockIdx.x & 7;
  const bool prefix = (int)(blockIdx.x >> 3) < gp;
  const int j = (int)(blockIdx.x >> 3) - (prefix ? 0 : gp);
  const bool direct = A.wa == nullptr;
  if (prefix) {
    const int id = x * gp + j;
    if (id >= np) return;
    const int tile = id % A.ntp, sp = id / A.ntp % A.nsp, hk = id / (A.ntp * A.nsp);
    const int len = prefix_len(A), r = range_keys(len, A.nsp, NW);
    const int k0 = min((long long)sp * r, (long long)len), k1 = min(k0 + r, len);
    if (k0 >= k1 && !direct) return;  // the join skips it too
    if constexpr (RTP == 0)
      wide_item<T, D, kWideRT, NW>(A, smem, hk, tile * 16 * kWideRT * NW, A.T * A.G, k0, k1, sp);
    else
      item<T, D, RTP, NW, false>(A, smem, hk, 0, tile * 16 * RTP, A.T * A.G, k0, k1, A.ptable, A.pblocks, 0, sp, direct);
  } else {
    const int id = x * go + j;
    if (id >= no) return;
    const int tile = id % A.nto, sp = id / A.nto % A.nso, hk = id / (A.nto * A.nso) % A.Hkv,
              b = id / (A.nto * A.nso) / A.Hkv;
    int tok0, n;
    seq_rows(A, b, tok0, n);
    const int row0 = tile * 16 * RTO;
    if (row0 >= n * A.G) return;
    const int len = own_len(A, b), r = range_keys(len, A.nso, NW);
    const int lim0 = len - n + 1;  // keys that the first new token sees
    const int last = min(len, lim0 + (min(row0 + 16 * RTO, n * A.G) - 1) / A.G);
    const int k0 = min((long long)sp * r, (long long)len), k1 = max(k0, min(k0 + r, last));
    if (k0 >= len && !direct) return;
    item<T, D, RTO, NW, true>(A, smem, hk, tok0, row0, n * A.G, k0, k1, A.tables + (long long)b * A.tstride,
                              A.max_blocks, lim0, A.nsp + sp, direct);
  }
}

// Join of a row's items: one wave a row, bounded by the read of the parts (17 us for 256 rows of 64 heads: 9 parts of
// 8.4 MB, 4.5 TB/s).  A row behind the last sequence, and a row that sees no key, is
// zero (lse -inf).  A row of a sequence that brings more tokens than the call allows is NaN.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(Args A, int nw) {
  constexpr int E = D / 64;
  const long long rows = (long long)A.T * A.Hq;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63, t = (int)(row / A.Hq);
  int b;
  bool over = false;
  if (A.cu) {
    b = __builtin_amdgcn_readfirstlane(seq_of_token(A.cu, A.B, t));
    if (b == A.B) b = -1;
    if (b >= 0) {
      int tok0, n;
      seq_rows(A, b, tok0, n);
      over = A.cu[b + 1] - tok0 > A.most;
      if (n == 0) b = -1;
    }
  } else {
    b = t < A.B ? t : -1;
  }
  const int pl = b >= 0 ? prefix_len(A) : 0, ol = b >= 0 ? own_len(A, b) : 0;
  const int rp = range_keys(pl, A.nsp > 0 ? A.nsp : 1, nw), ro = range_keys(ol, A.nso > 0 ? A.nso : 1, nw);
  const int ap = A.nsp > 0 ? (pl + rp - 1) / rp : 0, ao = A.nso > 0 ? (ol + ro - 1) / ro : 0;
  // the parts' statistics by lane, 64 at a time; then their sums, several loads in flight
  auto slot = [&](int s) { return (s < ap ? s : A.nsp + s - ap) * rows + row; };
  auto stats = [&](int s) { return s < ap + ao ? A.wml[slot(s)] : make_float2(-INFINITY, 0.f); };
  float M = -INFINITY;
  for (int s = lane; s - lane < ap + ao; s += 64) M = fmaxf(M, stats(s).x);
  M = wave_max(M);
  float L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s0 = 0; s0 < ap + ao; s0 += 64) {
    const float2 x = stats(s0 + lane);
    const float w = s0 + lane < ap + ao ? part_weight(x, M) : 0.f;
    L += x.y * w;
    const int n = min(64, ap + ao - s0);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
      float a[E];
      load_f<float, E>(A.wa + slot(s0 + j) * D + lane * E, a);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += a[e] * f;
    }
  }
  L = wave_sum(L);
  if (over) L = NAN;
  const float k = inverse_sum(L);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = L == 0.f ? 0.f : o[e] * k;
  store_f<T, E>(reinterpret_cast<T*>(A.out) + row * D + lane * E, o);
  if (A.lse && lane == 0) A.lse[row] = row_lse(M, L);
}

template <typename T, int D, int RTP, int RTO, int NW>
static hipError_t launch(const Args& A, hipStream_t st) {
  const long long np = (long long)A.Hkv * A.ntp * A.nsp, no = (long long)A.B * A.Hkv * A.nto * A.nso;
  const long long grid = 8 * ((np + 7) / 8 + (no + 7) / 8);
  if (np > 0x3fffffff || no > 0x3fffffff || grid > 0x7fffffff) return hipErrorInvalidValue;
  if (grid > 0) items_kernel<T, D, RTP, RTO, NW><<<(int)grid, NW * 64, 0, st>>>(A);
  if (A.wa) {
    const long long rows = (long long)A.T * A.Hq;
    join_kernel<T, D><<<(int)((rows + 3) / 4), 256, 0, st>>>(A, NW);
  }
  return hipGetLastError();
}

}  // namespace pfx
}  // namespace pa

using namespace pa::pfx;

// Head dims and waves of a block
static int pfx_nw(int D) { return D == 256 ? 4 : 8; }

// Row tiles of 16 an item holds: one where 16 rows hold them all, else as many as the registers do (the own
// items' masks take some of them)
static int pfx_rtp(long long rows, int D) { return rows <= 16 ? 1 : (D == 64 ? 4 : 2); }
// Whether the prefix items are wide: where more than half of a wide item's rows are there (fewer leave its waves
// idle).  Packed queries or a prefix alone go the same way: the join is always there with a prefix and own keys.
static bool pfx_wide(long long rows, int D) { return rows > 16 * kWideRT * pfx_nw(D) / 2; }
static int pfx_rto(long long rows, int D) { return rows <= 16 ? 1 : (D == 256 ? 1 : 2); }

// The cut of a call (`packed`: queries by offsets): out[0..3] = row tiles and key ranges (prefix, own), out[4] = slots (0: no workspace).
// `plen` / `own`: upper bounds of the prefix's and a sequence's length (the tables' capacity when the
// lengths are on the device).
PA_API int pa_prefix_attn_plan(int T, int B, int Hq, int Hkv, int D, int most, int packed, long long plen,
                                long long own, int* out) {
  if (T <= 0 || B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || most <= 0 || (D != 64 && D != 128 && D != 256))
    return (int)hipErrorInvalidValue;
  const long long G = Hq / Hkv, nw = pfx_nw(D);
  const int rtp = pfx_rtp((long long)T * G, D), rto = pfx_rto(most * G, D);
  const long long prow = pfx_wide((long long)T * G, D) ? 16 * kWideRT * nw : 16 * rtp;  // rows of a prefix item
  const long long ntp = (T * G + prow - 1) / prow, nto = (most * G + 16 * rto - 1) / (16 * rto);
  auto ranges = [&](long long len, long long items, long long target) -> long long {
    if (len <= 0) return 0;
    const long long cap = (len + 64 * nw - 1) / (64 * nw);  // two tiles a wave at least
    long long n = (target + items - 1) / items;
    // No block walks more than 8192 keys alone, as long as the parts take no more than 1 GiB for it: `len` is what the
    // table could hold, and with many new tokens a part for each 8192 keys of that would be more than there is
    // (65536 tokens of 64 heads of 128 with tables for 2^20: 280 GB).  Many new tokens fill the chip by their rows.
    const long long fits = (1ll << 28) / ((long long)T * Hq * (D + 2)), most_parts = fits < 1 ? 1 : fits;
    const long long least = (len + 8191) / 8192 < most_parts ? (len + 8191) / 8192 : most_parts;
    if (n < least) n = least;
    return n < 1 ? 1 : (n > cap ? cap : n);
  };
  const bool wide = pfx_wide((long long)T * G, D);
  out[0] = (int)ntp;
  if (wide) {
    // Beside own keys one round of blocks on 3/4 of the CUs, while the rest stream the own pages (256 sequences
    // behind 32768 shared keys and 500 .. 1500 of their own: 447 us; 508 with 256 blocks, 524 with 512, 571 with
    // 128); alone, two rounds.  At least 1024 keys a block: 8192 keys in ranges of 512 take 65 us beside 64
    // sequences, of 1024 61.
    const long long cap = (plen + 1023) / 1024, n = (own > 0 ? 192 : 512) / (Hkv * ntp);
    out[1] = plen <= 0 ? 0 : (int)(n < 1 ? 1 : (n > cap ? cap : n));
  } else {
    out[1] = (int)ranges(plen, Hkv * ntp, 512);  // two blocks a CU
  }
  out[2] = (int)nto;
  out[3] = (int)ranges(own, (long long)B * Hkv * nto, 512);
  if (out[1] + out[3] == 0) out[3] = 1;
  // one range for every row: written straight to the output; not with packed queries, of which some rows may
  // belong to no sequence and are the join's to clear
  out[4] = out[1] + out[3] == 1 && !packed && !(out[1] && wide) ? 0 : out[1] + out[3];
  return 0;
}

// ws: plan[4] * T * Hq * (D + 2) floats, partial outputs and their (max, sum)
PA_API int pa_prefix_attn(const void* q, const void* kc, const void* vc, long long qt, long long qh,
                          const long long* cstr, const int* tables, long long tstride, int max_blocks,
                          const int* ptable, int pblocks, const int* plen_dev, int plen, int num_blocks, int page,
                          const int* lens, const int* cu, void* out, float* lse, float* ws,
                          const int* plan, int T, int B, int Hq, int Hkv, int D, int most, float scale, int dt,
                          hipStream_t st) {
  if (T <= 0 || B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || page <= 0 || num_blocks < 0 || (dt != 1 && dt != 2) ||
      !(scale > 0.f) || cstr[2] < 0 || (!cu && T != B) || (plan[4] > 0 && !ws))
    return (int)hipErrorInvalidValue;
  Args A;
  A.q = (const uint16_t*)q; A.kc = (const uint16_t*)kc; A.vc = (const uint16_t*)vc;
  A.qt = qt; A.qh = qh; A.cb = cstr[0]; A.ch = cstr[1]; A.cr = cstr[2];
  A.tables = tables; A.tstride = tstride; A.max_blocks = max_blocks;
  A.ptable = ptable; A.pblocks = pblocks; A.plen_dev = plen_dev; A.plen = plen;
  A.lens = lens; A.cu = cu;
  A.out = (uint16_t*)out; A.lse = lse; A.wa = plan[4] > 0 ? ws : nullptr; A.wml = (float2*)(ws + (long long)plan[4] * T * Hq * D); A.most = most;
  A.num_blocks = num_blocks; A.page = page;
  A.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  A.T = T; A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.G = Hq / Hkv;
  A.ntp = plan[0]; A.nsp = plan[1]; A.nto = plan[2]; A.nso = plan[3];
  A.scale = scale * pa::fa::kLog2e;
  const int rtp = pfx_rtp((long long)T * A.G, D), rto = pfx_rto((long long)most * A.G, D);
  const bool wide = A.nsp > 0 && pfx_wide((long long)T * A.G, D);
#define PA_PFX(TT, DD, RP, RO, NW)                                               \
  if (D == DD) {                                                                 \
    if (wide && rto > 1) return (int)launch<TT, DD, 0, RO, NW>(A, st);           \
    if (wide) return (int)launch<TT, DD, 0, 1, NW>(A, st);                       \
    if (RO > 1 && rto > 1) return (int)launch<TT, DD, RP, RO, NW>(A, st);        \
    if (rtp > 1) return (int)launch<TT, DD, RP, 1, NW>(A, st);                   \
    return (int)launch<TT, DD, 1, 1, NW>(A, st);                                 \
  }
#define PA_PFX_T(TT)           \
  PA_PFX(TT, 64, 4, 2, 8)      \
  PA_PFX(TT, 128, 2, 2, 8)     \
  PA_PFX(TT, 256, 2, 1, 4)
  if (dt == 1) {
    PA_PFX_T(pa::bf16_t)
  } else {
    PA_PFX_T(pa::f16_t)
  }
#undef PA_PFX_T
#undef PA_PFX
  return (int)hipErrorInvalidValue;
}
