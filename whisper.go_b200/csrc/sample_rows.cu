// sample_rows.cu — drawing tokens with temperature, top-k, top-p and min-p
// from given random numbers (wg_sample_rows).
//
// With w_i = exp((x_i - max x) / T), every filter keeps a prefix of the row in
// descending order (lower index first among equals), so the kept set is one
// cut: the elements above a value, and the first J of those equal to it.
//
// Which token a random number falls on is decided by sums of up to V weights,
// so the weights that decide are evaluated in 64-bit floats and summed as
// integers in units of 2^-45 (at most 2^18 * 2^45 for a row): sums are exact,
// free of any order, and off by less than V * 2^-46 of the largest weight
// from the real ones. The sum under the log-prob is fp32.
//
// A cluster of C CTAs takes a row; each holds its slice in shared memory as
// fp32, so the row is read from memory once and every later pass is over
// shared memory. Nothing is ordered but a short list:
//  1. a histogram of counts over SR_BINS equal steps of the logit below the
//     maximum (one shared atomic an element) gives the bin of the top-k cut,
//     and with the masses of the heavy elements and count * exp(middle) for
//     the light bins the likely bin of the top-p cut;
//  2. where the bins that can be kept hold at most SR_LIST elements (as a
//     rule: a nucleus, a top-k, a min-p set), those go to rank 0 in index
//     order, which puts them into their bins, orders each bin by counting
//     (320 rows: nucleus 111 -> 102 us against a sort of the list, k 200 80 ->
//     70) and finishes alone. Its peers leave then, except under top-p without
//     top-k, which may need the exact mass of the rest of the row (k 50 84 ->
//     66 us, with the lists pushed rather than fetched);
//  3. else the few bins that hold the cut go to rank 0, which orders them and
//     reads the cut off their running counts or exact masses (such rows 27 us
//     alone, 38 to 47 with descents); where those bins hold too many, under
//     both top-k and top-p, or where the likely bin was wrong, it is pinned by
//     descents over the order-preserving bit patterns of the logits, 9 bits a
//     pass, with exact counts and masses. The draw then walks cluster rank ->
//     thread -> element over the kept masses of each thread's consecutive
//     elements;
//  4. rows without filters are walked over their fp32 weights first, and over
//     exact ones only where the number falls too near an element's edge for
//     the bounds on those (320 such rows 81 -> 58 us).
//
// What bounds it: latency. Of a row's ~15 us the load is 1.5, the exchanges of
// the cluster (maxima, histogram, list) ~4, rank 0's ordering and draw ~3; the
// SMs hold 111 rows of 51866 at once (three CTAs of 75 KB each), and most
// stalls are barriers. 64-bit weights of a whole row would cost as much again,
// so top-p asks for them only where bounds on the fp32 sum do not settle the cut
// (3 % of such rows), and with eleven operations each. Measured (a pass): one
// row of 51865 fp32 15 us (24 where no short list holds the kept set), 48 of
// 51864 f16 25 us, 320 of 51866 fp32 76 us = 0.87 TB/s; 61 us with a top-k in
// the place of the nucleus rows, of which two in 54 have no short list and may
// come last. One CTA a row, streaming the row from L2 in every pass: top-k 81 us
// at 320 rows against 67, 53 at one row against 14.
#include <cooperative_groups.h>

#include <cstddef>
#include <mutex>

#include "kernels.cuh"
#include "ops.cuh"

namespace wg {
namespace {

namespace cg = cooperative_groups;

constexpr int SR_THREADS = 256;
constexpr int SR_WARPS = SR_THREADS / 32;
constexpr int SR_BPT = 2;                 // bins a thread
constexpr int SR_BINS = SR_BPT * SR_THREADS;  // of the first histogram
constexpr int SR_SUB = SR_BPT * SR_THREADS;   // of a descent (9 bits)
constexpr int SR_EPT = 4;                 // candidates a thread
constexpr int SR_LIST = SR_EPT * SR_THREADS;  // that rank 0 can finish alone
constexpr int SR_MAX_CLUSTER = 8;
constexpr int SR_TABLE = 256;
constexpr float SR_SPAN = 40.f;           // logits that far below the maximum share the last bin
constexpr float SR_HEAVY = 1.f / 1024.f;  // weights above it are summed in the first histogram
constexpr double SR_STEP = -0.69314718055994530942 / SR_TABLE;  // ln of a table step
constexpr float SR_OCTAVES = 46.5f;       // weights below 2^-46.5 are 0 in those units
constexpr int SR_MAX_V = 1 << 18;
constexpr int SR_PAD = 8;                 // a slice may start up to 7 elements into its 16 bytes
enum { SR_DONE = 0, SR_EXACT = 1, SR_WHOLE = 2 };  // what rank 0 still needs: nothing, the exact mass, the whole row
typedef unsigned long long u64;

// Unsigned keys in the order of the values (-0 with +0); 0 is no value's key.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Shared {
  // per rank, pushed by every rank to every rank before a cluster barrier (a
  // remote store costs its sender nothing, a remote load is ~0.3 us of waiting)
  float mx[SR_MAX_CLUSTER], mn[SR_MAX_CLUSTER];
  double sum[SR_MAX_CLUSTER];                      // the slice's fp32 weights below 1, threads' sums added in 64 bits
  unsigned ones[SR_MAX_CLUSTER];                   // and how many are 1 (the maxima)
  int first[SR_MAX_CLUSTER];                       // lowest index of the slice that holds the maximum
  u64 all[SR_MAX_CLUSTER], over[SR_MAX_CLUSTER];   // exact sums of the slice: whole, and above the likely bins
  u64 kept[SR_MAX_CLUSTER];                        // kept mass without ties
  unsigned ties[SR_MAX_CLUSTER];                   // elements equal to the cut
  int drawn;                                       // a rank has drawn the row's token
  unsigned listed;                                 // at rank 0: elements of the cut's bins
  uint32_t cut_key;                                // from rank 0: the cut that their order gives, where cut_ties > 0
  unsigned cut_ties;
  int again;                                       // from rank 0: SR_DONE, SR_EXACT or SR_WHOLE
  // read by peers after a cluster barrier
  alignas(16) uint2 hist[SR_BINS];                 // count, mass of the heavy ones (2^-16 units)
  union alignas(16) {
    uint4 sub[2][SR_SUB];  // descents: count, mass in three 15-bit digits (summed in 32 bits: for < 2^17 elements)
    struct {
      int2 xi[SR_LIST];    // rank 0: the row's candidates in index order, pushed by every rank (logit, index)
      u64 order[SR_LIST];  // the same to order, then their kept masses in index order
    } list;
    struct {
      u64 mass[SR_THREADS];       // kept mass of each thread's elements
      unsigned ties[SR_THREADS];  // and how many equal the cut
    } part;
  };
  // this CTA's own
  double pow2[SR_TABLE];  // 2^(-j / 256)
  u64 red_m[SR_WARPS], red_o[SR_WARPS];
  unsigned red_c[SR_WARPS];
  float red_f[2][SR_WARPS];
  int found[2];
  u64 found_m;
  unsigned found_c;
};
static_assert(SR_BPT == 2 && offsetof(Shared, hist) % 16 == 0, "a thread's bins are one uint4");
static_assert(offsetof(Shared, sub) % 16 == 0, "descent bins are read as uint4");
constexpr int SR_HEAD = (int)((sizeof(Shared) + 15) / 16 * 16);  // the slice begins here
constexpr int SR_SMEM_MAX = 227 * 1024;

// Asked for anew where they are used: a pointer that went through memory would
// be a generic one, and its accesses too.
__device__ __forceinline__ Shared& shared_part() {
  extern __shared__ __align__(16) uint8_t dyn[];
  return *reinterpret_cast<Shared*>(dyn);
}
__device__ __forceinline__ float* shared_slice() {
  extern __shared__ __align__(16) uint8_t dyn[];
  return reinterpret_cast<float*>(dyn + SR_HEAD);
}
static_assert(SR_SMEM_MAX / (16 * SR_THREADS) <= 64, "a thread's groups of four are bits of one word");

// The weight of a logit: the definition's 64-bit value by argument reduction.
// With y = 256 (max - x) / (T ln 2) = n + r, n the nearest integer,
// w = 2^-(n >> 8) * 2^-((n & 255) / 256) * exp(-r ln 2 / 256): the exponent, a
// table, and a Taylor series (|r ln 2 / 256| <= 0.00136: four terms leave 4e-17).
struct Weigh {
  double mx, c;  // c = 256 / (T ln 2)
  // w = v * 2^-oct
  __device__ __forceinline__ double value(float x, int* oct) const {
    const double magic = 6755399441055744.0;  // 2^52 + 2^51: a sum's low word is the nearest integer
    const double d = mx - (double)x, shifted = fma(d, c, magic);
    const int n = __double2loint(shifted);
    const double r = fma(d, c, magic - shifted);
    constexpr double a1 = SR_STEP, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4;
    double p = fma(r, a4, a3);
    p = fma(p, r, a2);
    p = fma(p, r, a1);
    p = fma(p, r, 1.0);
    *oct = n >> 8;
    return shared_part().pow2[n & (SR_TABLE - 1)] * p;
  }
  // w in units of 2^-45: v * 2^(45 - oct) + 2^52 leaves the rounded integer in the low 52 bits
  static __device__ __forceinline__ u64 fixed(double v, int oct) {
    const double scale = __hiloint2double((1023 + 45 - oct) << 20, 0);
    return (u64)__double_as_longlong(fma(v, scale, 4503599627370496.0)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 fixed_of(float x) const {
    int oct;
    const double v = value(x, &oct);
    return fixed(v, oct);
  }
  // for octaves below 1022
  __device__ __forceinline__ bool at_least(float x, double least) const {
    int oct;
    const double v = value(x, &oct);
    return v * __hiloint2double((1023 - oct) << 20, 0) >= least;
  }
  // in those units, 0 where w < least
  __device__ __forceinline__ u64 fixed_from(float x, double least) const {
    int oct;
    const double v = value(x, &oct);
    return v * __hiloint2double((1023 - oct) << 20, 0) >= least ? fixed(v, oct) : 0;
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Inclusive scans over the CTA of a mass and a count; *tm, *tc: the totals.
__device__ __forceinline__ void block_scan(Shared& sh, u64& m, unsigned& c, u64* tm, unsigned* tc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(0xffffffffu, m, o);
    const unsigned b = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) { m += a; c += b; }
  }
  __syncthreads();  // earlier readers of red_* are done
  if (lane == 31) { sh.red_m[warp] = m; sh.red_c[warp] = c; }
  __syncthreads();
  u64 am = 0, pm = 0;
  unsigned ac = 0, pc = 0;
#pragma unroll
  for (int w = 0; w < SR_WARPS; w++) {
    if (w == warp) { pm = am; pc = ac; }
    am += sh.red_m[w];
    ac += sh.red_c[w];
  }
  m += pm;
  c += pc;
  *tm = am;
  *tc = ac;
}

struct Cut {
  uint32_t key;   // elements above it are kept (0: every element)
  unsigned ties;  // and so many of those equal to it, in index order
};

template <typename T>
__device__ __forceinline__ T* peer(T* p, int rank, int C) {
  return C > 1 ? cg::this_cluster().map_shared_rank(p, rank) : p;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier(int C) {
  if (C > 1) cg::this_cluster().sync();
  else __syncthreads();
}

// What a row's passes share: kept in registers by the kernel, handed over in
// memory to the passes that few rows need (in one body they cost the others
// registers: one row 15.1 us, 15.9 in one body; 320 with a top-k 67 and 71).
struct Row {
  wg_sample s;
  int C, rank, r, per;
  int first_i;  // index of the thread's first element
  int slice;
  float mx, span, bin_scale, t1, c2, c2_lo, deep, u;
  Weigh wt;
  int k;
  float top_p;
  double least;  // min-p
  bool by_k, by_p, by_m;

  // this thread's consecutive elements
  __device__ __forceinline__ const float4* mine() const {
    return reinterpret_cast<const float4*>(shared_slice() + threadIdx.x * per);
  }
  // f(x[4], i) over the thread's elements, i the place of the first of the four
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 1
    for (int i = 0; i < per; i += 4) {
      const float4 v = mine()[i / 4];
      const float x[4] = {v.x, v.y, v.z, v.w};
      f(x, i);
    }
  }
  __device__ __forceinline__ float octaves(float x) const {
    const float d = fmaxf(x - mx, deep);
    return fmaf(d, c2, d * c2_lo);
  }
  // nearest bin, the last one for everything further down (2^23 + b holds b in its low bits)
  __device__ __forceinline__ float bin_bits(float x) const { return fminf((mx - x) * bin_scale, (float)(SR_BINS - 1)) + 8388608.f; }
  __device__ __forceinline__ int bin_of(float x) const { return __float_as_int(bin_bits(x)) & (SR_BINS - 1); }
  __device__ __forceinline__ bool light(float x) const { return !((mx - x) * c2 < SR_OCTAVES); }
  __device__ __forceinline__ u64 weight(float x) const { return light(x) ? (u64)0 : wt.fixed_of(x); }
  __device__ __forceinline__ u64 weight_kept(float x) const {
    if (u == 0.f) return first_kept(x);
    return light(x) ? (u64)0 : by_m ? wt.fixed_from(x, least) : wt.fixed_of(x);
  }
  // The number 0 falls on the first token that stays, however small its weight:
  // all count alike. (min_p, an fp32 number, is at least 2^-149.)
  __device__ __forceinline__ u64 first_kept(float x) const {
    return x > -INFINITY && (!by_m || ((mx - x) * c2 < 160.f && wt.at_least(x, least)));
  }
  __device__ __forceinline__ void finish(int token, float x) const {
    s.tokens[r] = token;
    if (s.logprobs) {
      const Shared& sh = shared_part();
      double z = 0;
      unsigned n1 = 0;
      for (int q = 0; q < C; q++) {
        z += sh.sum[q];
        n1 += sh.ones[q];
      }
      s.logprobs[r] = (x - mx) / t1 - (logf((float)n1) + log1pf((float)z / (float)n1));
    }
  }
  // first running mass above u * mass
  __device__ __forceinline__ u64 draw(u64 mass) const {
    const double at = (double)u * (double)mass;
    const u64 goal = at < (double)mass ? (u64)at + 1 : mass;
    return goal > mass ? mass : goal;
  }
  // the running mass that top-p asks for
  __device__ __forceinline__ u64 share(u64 mass) const {
    const double want = ceil((double)top_p * (double)mass);
    const u64 goal = want >= 1.0 ? (u64)want : 1;
    return goal > mass ? mass : goal;
  }
  // The fp32 weights 2^-y, and any sum of them, are off by at most this share of
  // their whole sum z: ex2.approx 2^-22; three roundings of y, each 2^-24 of it,
  // and the mean of y over the mass is at most log2 V - log2 z (an entropy);
  // per / 4 additions in fp32; 2^-24 for what the exact units round off (V * 2^-46)
  __device__ __forceinline__ float off_by(float z) const {
    return (6.f + 2.1f * fmaxf(0.f, log2f((float)s.V) + 0.01f - log2f(z)) + (float)(per / 4)) * (1.f / 16777216.f);
  }

  __device__ void long_passes(int kbin, int pbin, unsigned kabove) const;
};

// Rows whose kept set no short list holds, and rows without filters that the
// fp32 weights do not decide.
__device__ __forceinline__ void Row::long_passes(int kbin, int pbin, unsigned kabove) const {
  Shared& sh = shared_part();
  const float* xs = shared_slice();
  const float4* mine = this->mine();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 all;
  // ---- the cut
  // By a list, once a row: the elements of bins ba..bb go to rank 0 in any order.
  auto inside = [&](float x, int ba, int bb) {
    const int b = bin_of(x);
    return b >= ba && b <= bb && x > -INFINITY;
  };
  auto push_bins = [&](int ba, int bb, u64 fours, unsigned hits) {
    const unsigned own_hits = hits;
    unsigned hits_t;
    u64 none = 0, none_t;
    block_scan(sh, none, hits, &none_t, &hits_t);
    if (tid == 0) sh.found[0] = (int)atomicAdd(peer(&sh.listed, 0, C), hits_t);
    __syncthreads();
    unsigned at = (unsigned)sh.found[0] + hits - own_hits;
    u64* to = peer(sh.list.order, 0, C);
    for (; fours; fours &= fours - 1) {
      const int i = __ffsll((long long)fours) - 1;
      const float4 v = mine[i];
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (inside(x[j], ba, bb)) {
          if (at < SR_LIST) to[at] = ((u64)key_of(x[j]) << 32) | (0xffffffffu - (unsigned)(first_i + 4 * i + j));
          at++;
        }
    }
  };
  // Rank 0 orders them (SR_BINS parts of their bins, then by counting inside a
  // part) and tells the element where the running count (or mass) reaches
  // `target`. False where it does not, or where there are more than SR_LIST.
  // A cluster barrier lies between the pushes and this.
  auto cut_of_list = [&](bool mass, u64 target, int ba, int bb, u64 above, Cut* out) -> bool {
    const int total = (int)sh.listed;
    if (rank == 0 && total <= SR_LIST) {
      const float fine = (float)SR_BINS / (float)(bb - ba + 1);
      auto part_of = [&](u64 v) {  // falls with the logit
        const float at = ((mx - of_key((uint32_t)(v >> 32))) * bin_scale - ((float)ba - 0.5f)) * fine;
        return (int)fminf(fmaxf(at, 0.f), (float)(SR_BINS - 1));
      };
      unsigned* begin = reinterpret_cast<unsigned*>(sh.hist);  // read last before the barrier above
      u64* by_part = reinterpret_cast<u64*>(sh.list.xi);
      begin[SR_BPT * tid] = begin[SR_BPT * tid + 1] = 0;
      __syncthreads();
      for (int i = tid; i < total; i += SR_THREADS) atomicAdd(&begin[part_of(sh.list.order[i])], 1u);
      __syncthreads();
      const unsigned n0 = begin[SR_BPT * tid], n1 = begin[SR_BPT * tid + 1];
      unsigned c = n0 + n1, tc;
      u64 m = 0, tm;
      block_scan(sh, m, c, &tm, &tc);
      begin[SR_BPT * tid] = c - n0 - n1;
      begin[SR_BPT * tid + 1] = c - n1;
      __syncthreads();
      for (int i = tid; i < total; i += SR_THREADS) {
        const u64 v = sh.list.order[i];
        by_part[atomicAdd(&begin[part_of(v)], 1u)] = v;
      }
      __syncthreads();  // a part begins where the one before it ended
      for (int e = tid; e < total; e += SR_THREADS) {
        const u64 v = by_part[e];
        const int b = part_of(v), from = b ? (int)begin[b - 1] : 0, end = (int)begin[b];
        int at = from;
        for (int i = from; i < end; i++) at += by_part[i] > v;
        sh.list.order[at] = v;
      }
      __syncthreads();
      const int each_t = (total + SR_THREADS - 1) / SR_THREADS, e0 = each_t * tid;
      u64 f[SR_EPT] = {};
#pragma unroll
      for (int j = 0; j < SR_EPT; j++) {
        if (j < each_t && e0 + j < total) f[j] = mass ? weight(of_key((uint32_t)(sh.list.order[e0 + j] >> 32))) : 1;
        m += f[j];
      }
      const u64 own_mass = m;
      block_scan(sh, m, c, &tm, &tc);
      u64 run = above + m - own_mass;
#pragma unroll
      for (int j = 0; j < SR_EPT; j++) {
        if (f[j] && run < target && target <= run + f[j]) {
          const int e = e0 + j;
          const uint32_t key = (uint32_t)(sh.list.order[e] >> 32);
          unsigned ties = 1;
          while ((int)ties <= e && (uint32_t)(sh.list.order[e - ties] >> 32) == key) ties++;
          for (int q = 0; q < C; q++) {
            peer(&sh, q, C)->cut_key = key;
            peer(&sh, q, C)->cut_ties = ties;
          }
        }
        run += f[j];
      }
    }
    cluster_barrier(C);
    if (!sh.cut_ties) return false;
    out->key = sh.cut_key;
    out->ties = sh.cut_ties;
    return true;
  };
  int level = 0;  // descents so far: their buffers alternate
  auto clear = [&]() {
    for (int i = tid; i < SR_SUB; i += SR_THREADS) sh.sub[level & 1][i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  };
  // The cut where the running count (or mass) in descending order reaches
  // `target`, known to lie in bins ba..bb, above which there are `above`;
  // among the elements inside `in`. False where it does not lie there.
  auto descend = [&](const Cut& in, bool mass, u64 target, int ba, int bb, u64 above, Cut* out) -> bool {
    // keys that the bins can hold (a hundredth of a bin and a few ulps around them)
    const float w = span / (float)(SR_BINS - 1), slack = 0.01f * w + 1e-6f * fabsf(mx);
    uint32_t klo = bb >= SR_BINS - 1 ? 0u : key_of(mx - ((float)bb + 0.5f) * w - slack);
    uint32_t khi = ba <= 0 ? key_of(mx) : key_of(fminf(mx, mx - ((float)ba - 0.5f) * w + slack));
    for (;;) {
      int shift = 0;
      while (((khi - klo) >> shift) >= (uint32_t)SR_SUB) shift++;
      uint4* sub = sh.sub[level & 1];
      auto put = [&](float x, uint32_t key, unsigned count) {
        const int b = bin_of(x);
        if (b < ba || b > bb) return;
        unsigned* to = &sub[(key - klo) >> shift].x;
        atomicAdd(to, count);
        if (mass) {
          const u64 f = weight(x);
          atomicAdd(to + 1, (unsigned)(f & 0x7fffu) * count);
          atomicAdd(to + 2, (unsigned)(f >> 15 & 0x7fffu) * count);
          atomicAdd(to + 3, (unsigned)(f >> 30) * count);
        }
      };
      each([&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t key = key_of(x[j]);
          if (key >= klo && key <= khi && key > in.key) put(x[j], key, 1u);
        }
      });
      // the ties of `in`, dealt over the ranks: a digit's sum holds a slice's elements and as many ties
      if (in.ties && tid == 0 && in.key >= klo && in.key <= khi) {
        const unsigned part = (in.ties + C - 1) / C, from = min(in.ties, part * rank);
        put(of_key(in.key), in.key, min(in.ties, from + part) - from);
      }
      cluster_barrier(C);
      // sub-bins in descending order: thread t has SUB - 1 - BPT * t and the next below
      unsigned c1[SR_BPT] = {}, c = 0, tc;
      u64 m1[SR_BPT] = {}, m = 0, tm;
#pragma unroll
      for (int q = 0; q < SR_MAX_CLUSTER; q++)
        if (q < C) {
#pragma unroll
          for (int b = 0; b < SR_BPT; b++) {
            const uint4 v = peer(sub, q, C)[SR_SUB - 1 - SR_BPT * tid - b];
            c1[b] += v.x;
            m1[b] += (u64)v.y + ((u64)v.z << 15) + ((u64)v.w << 30);
          }
        }
      level++;
      for (int i = tid; i < SR_SUB; i += SR_THREADS) sh.sub[level & 1][i] = make_uint4(0u, 0u, 0u, 0u);  // read last before the barrier above
#pragma unroll
      for (int b = 0; b < SR_BPT; b++) {
        c += c1[b];
        m += m1[b];
      }
      const unsigned c_own = c;
      const u64 m_own = m;
      block_scan(sh, m, c, &tm, &tc);
      if (tid == 0) sh.found[0] = -1;
      __syncthreads();
      u64 run = above + (mass ? m - m_own : (u64)(c - c_own));
#pragma unroll
      for (int b = 0; b < SR_BPT; b++) {
        const u64 one = mass ? m1[b] : (u64)c1[b];
        if (c1[b] && run < target && run + one >= target) {
          sh.found[0] = SR_SUB - 1 - SR_BPT * tid - b;
          sh.found_m = run;
          sh.found_c = c1[b];
        }
        run += one;
      }
      __syncthreads();
      const int sel = sh.found[0];
      if (sel < 0) return false;
      above = sh.found_m;
      klo += (uint32_t)sel << shift;
      khi = min(khi, klo + ((1u << shift) - 1u));
      if (shift == 0) {
        const u64 each_w = mass ? weight(of_key(klo)) : 1;
        u64 j = each_w ? (target - above + each_w - 1) / each_w : sh.found_c;
        if (j > sh.found_c) j = sh.found_c;
        out->key = klo;
        out->ties = (unsigned)j;
        return true;
      }
    }
  };

  Cut cut{0u, 0u};
  if (by_k) {
    const Cut every{0u, 0u};
    u64 fours = 0;
    unsigned hits = 0;
    for (int i = 0; i < per / 4; i++) {
      const float4 v = mine[i];
      const int h = inside(v.x, kbin, kbin) + inside(v.y, kbin, kbin) + inside(v.z, kbin, kbin) + inside(v.w, kbin, kbin);
      if (h) fours |= 1ull << i;
      hits += h;
    }
    push_bins(kbin, kbin, fours, hits);
    cluster_barrier(C);
    if (!cut_of_list(false, (u64)k, kbin, kbin, kabove, &cut)) {
      clear();
      if (!descend(every, false, (u64)k, kbin, kbin, kabove, &cut))
        descend(every, false, (u64)k, 0, SR_BINS - 1, 0, &cut);
    }
  }
  if (by_p) {
    // exact masses: of the top-k, and of what lies above the likely bins; the list in the same pass
    const int ba = max(0, pbin - 1), bb = min(SR_BINS - 1, pbin + 1);
    u64 over = 0, fours = 0;
    unsigned hits = 0;
    all = 0;
    each([&](const float (&x)[4], int i) {
      int h = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const u64 f = key_of(x[j]) > cut.key ? weight(x[j]) : 0;
        all += f;
        over += bin_of(x[j]) < ba ? f : 0;
        h += inside(x[j], ba, bb);
      }
      if (h) fours |= 1ull << (i / 4);
      hits += h;
    });
    if (!by_k) push_bins(ba, bb, fours, hits);
    all = warp_sum64(all);
    over = warp_sum64(over);
    __syncthreads();  // red_m has been read
    if (lane == 0) { sh.red_m[warp] = all; sh.red_o[warp] = over; }
    __syncthreads();
    if (warp == 0) {
      all = warp_sum64(lane < SR_WARPS ? sh.red_m[lane] : 0);
      over = warp_sum64(lane < SR_WARPS ? sh.red_o[lane] : 0);
      if (lane < C) {
        peer(sh.all, lane, C)[rank] = all;
        peer(sh.over, lane, C)[rank] = over;
      }
    }
    cluster_barrier(C);
    all = over = 0;
    for (int q = 0; q < C; q++) {
      all += sh.all[q];
      over += sh.over[q];
    }
    if (cut.ties) {
      const float x = of_key(cut.key);
      const u64 f = (u64)cut.ties * weight(x);
      all += f;
      if (bin_of(x) < ba) over += f;
    }
    const u64 goal = share(all);
    const Cut in = cut;
    if (by_k || !cut_of_list(true, goal, ba, bb, over, &cut)) {
      clear();
      if (over >= goal || !descend(in, true, goal, ba, bb, over, &cut))
        descend(in, true, goal, 0, SR_BINS - 1, 0, &cut);  // the guess was wrong: over the whole row
    }
  }

  // ---- the kept mass of every thread's elements
  {
    u64 m = 0;
    unsigned e = 0;
    each([&](const float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t key = key_of(x[j]);
        e += key == cut.key;
        if (key > cut.key) m += weight_kept(x[j]);
      }
    });
    // `part` shares the descents' memory: that was read last before a cluster barrier only
    // where a rank waits for its peers once more
    if (by_k || by_p) cluster_barrier(C);
    sh.part.mass[tid] = m;
    sh.part.ties[tid] = e;
    m = warp_sum64(m);
    e = __reduce_add_sync(0xffffffffu, e);
    __syncthreads();
    if (lane == 0) { sh.red_m[warp] = m; sh.red_c[warp] = e; }
    __syncthreads();
    if (warp == 0) {
      m = warp_sum64(lane < SR_WARPS ? sh.red_m[lane] : 0);
      e = __reduce_add_sync(0xffffffffu, lane < SR_WARPS ? sh.red_c[lane] : 0u);
      if (lane == 0) {
        peer(sh.kept, 0, C)[rank] = m;
        peer(sh.ties, 0, C)[rank] = e;
      }
    }
  }
  cluster_barrier(C);
  if (rank == 0) {
    // ties at the cut: their common weight, 0 where min-p drops them
    const u64 tie = cut.ties ? weight_kept(of_key(cut.key)) : 0;
    u64 mass = 0;
    unsigned left = cut.ties;
    for (int q = 0; q < C; q++) {
      const unsigned e = min(left, sh.ties[q]);
      mass += sh.kept[q] + e * tie;
      left -= e;
    }
    u64 goal = draw(mass);
    // cluster rank
    int q = 0;
    left = cut.ties;
    for (; q < C - 1; q++) {
      const unsigned e = min(left, sh.ties[q]);
      const u64 here = sh.kept[q] + e * tie;
      if (goal <= here) break;
      goal -= here;
      left -= e;
    }
    Shared* o = peer(&sh, q, C);
    // thread: running mass with the running number of ties, of which `left` stay
    const u64 m1 = o->part.mass[tid];
    const unsigned e1 = o->part.ties[tid];
    u64 m = m1, tm;
    unsigned e = e1, tc;
    if (tid == 0) { sh.found[0] = 0; sh.found_m = 1; sh.found_c = 0; }
    block_scan(sh, m, e, &tm, &tc);
    const u64 upto = m + min(e, left) * tie, before = m - m1 + min(e - e1, left) * tie;
    if (upto >= goal && before < goal) {
      sh.found[0] = tid;
      sh.found_m = goal - before;
      sh.found_c = left - min(e - e1, left);  // ties still to keep in it
    }
    __syncthreads();
    if (warp == 0) {
      const int owner = sh.found[0];
      goal = sh.found_m;
      left = sh.found_c;
      // element: the owner's consecutive ones, 32 at a time
      const int es = dt_bytes(s.dtype), vec = 16 / es, qc0 = min(s.V, q * slice);
      const uint8_t* qsrc = reinterpret_cast<const uint8_t*>(s.logits) + ((int64_t)r * s.ld + qc0) * es;
      const int qi = qc0 - (int)((reinterpret_cast<uintptr_t>(qsrc) / es) % vec) + owner * per;
      const float* qx = peer(xs, q, C) + owner * per;
      for (int i0 = 0; i0 < per; i0 += 32) {
        const int i = i0 + lane;
        const float x = i < per ? qx[i] : -INFINITY;
        const uint32_t key = key_of(x);
        const bool is_tie = key == cut.key;
        const unsigned ties = __ballot_sync(0xffffffffu, is_tie);
        u64 f = 0;
        if (is_tie) f = (unsigned)__popc(ties & ((1u << lane) - 1u)) < left ? tie : 0;
        else if (key > cut.key) f = weight_kept(x);
        u64 run = f;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const u64 v = __shfl_up_sync(0xffffffffu, run, d);
          if (lane >= d) run += v;
        }
        if (f && run >= goal && run - f < goal) finish(qi + i, x);
        const u64 here = __shfl_sync(0xffffffffu, run, 31);
        if (goal <= here) break;
        goal -= here;
        left -= min(left, (unsigned)__popc(ties));
      }
    }
  }
  cluster_barrier(C);  // rank 0 has read its peers
}

__device__ __noinline__ void finish_long(const Row& given, int kbin, int pbin, unsigned kabove) {
  const Row row = given;  // into registers
  row.long_passes(kbin, pbin, kabove);
}

// grid (C * R), cluster (C, 1, 1); dynamic shared memory: Shared, then the
// slice: `per` (4 times an odd number: no bank conflicts) consecutive elements
// for each thread, padded with -inf
__global__ void __launch_bounds__(SR_THREADS, 3) sample_rows_kernel(const wg_sample s, int C, int per) {
  Shared& sh = shared_part();
  float* xs = shared_slice();
  pdl_trigger();
  if (C > 1) cluster_arrive();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % C, r = blockIdx.x / C;
  const int slice = per * SR_THREADS - SR_PAD;
  const int c0 = min(s.V, rank * slice), n = min(s.V, c0 + slice) - c0;
  const float T = s.temperature ? s.temperature[r] : 1.f;
  const int k = s.top_k ? s.top_k[r] : 0;
  const float top_p = s.top_p ? s.top_p[r] : 1.f, min_p = s.min_p ? s.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < s.V, by_p = !(top_p >= 1.f), by_m = min_p > 0.f;
  // rows where only the first maximum can stay
  const bool top1 = !(T > 0.f) || k == 1 || !(top_p > 0.f) || !(min_p <= 1.f);
  const bool need_bins = !top1 && (by_k || by_p || by_m);
  for (int i = tid; i < SR_BINS; i += SR_THREADS) sh.hist[i] = make_uint2(0u, 0u);
  if (tid == 0) {
    sh.again = sh.drawn = 0;
    sh.listed = sh.cut_ties = 0;
  }

  // ---- the slice into shared memory, 16-byte loads between its ragged ends;
  // it starts at the address's place in 16 bytes, so both sides are aligned
  const int es = dt_bytes(s.dtype), vec = 16 / es;
  const uint8_t* src = reinterpret_cast<const uint8_t*>(s.logits) + ((int64_t)r * s.ld + c0) * es;
  const int lead = (int)((reinterpret_cast<uintptr_t>(src) / es) % vec);
  float mx = -INFINITY, mn = INFINITY;
  {
    auto clean = [&](float x) {
      x = x != x ? -INFINITY : x;
      mx = fmaxf(mx, x);
      mn = fminf(mn, x == -INFINITY ? INFINITY : x);  // the least finite one
      return x;
    };
    const int head = min(n, (vec - lead) % vec), body = (n - head) / vec, tail = n - head - body * vec;
    if (tid < lead) xs[tid] = -INFINITY;
    for (int i = lead + n + tid; i < per * SR_THREADS; i += SR_THREADS) xs[i] = -INFINITY;
    if (tid < head) xs[lead + tid] = clean(dt_load(src, tid, s.dtype));
    if (tid < tail) xs[lead + n - tail + tid] = clean(dt_load(src, n - tail + tid, s.dtype));
    const uint4* v = reinterpret_cast<const uint4*>(src + head * es);
    float4* d = reinterpret_cast<float4*>(xs + lead + head);
    constexpr int U = 4;  // loads in flight per thread
    for (int i0 = tid; i0 < body; i0 += U * SR_THREADS) {
      uint4 w[U];
#pragma unroll
      for (int j = 0; j < U; j++) w[j] = i0 + j * SR_THREADS < body ? __ldg(v + i0 + j * SR_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < U; j++) {
        const int i = i0 + j * SR_THREADS;
        if (i >= body) break;
        if (s.dtype == WG_DT_F32) {
          d[i] = make_float4(clean(__uint_as_float(w[j].x)), clean(__uint_as_float(w[j].y)),
                             clean(__uint_as_float(w[j].z)), clean(__uint_as_float(w[j].w)));
        } else {
          const float2 a = dt_unpack2(s.dtype, w[j].x), b = dt_unpack2(s.dtype, w[j].y);
          const float2 e = dt_unpack2(s.dtype, w[j].z), f = dt_unpack2(s.dtype, w[j].w);
          d[2 * i] = make_float4(clean(a.x), clean(a.y), clean(b.x), clean(b.y));
          d[2 * i + 1] = make_float4(clean(e.x), clean(e.y), clean(f.x), clean(f.y));
        }
      }
    }
  }
  for (int i = tid; i < SR_TABLE; i += SR_THREADS) sh.pow2[i] = exp2(-(double)i / SR_TABLE);
  mx = warp_max(mx);
  mn = -warp_max(-mn);
  if (lane == 0) { sh.red_f[0][warp] = mx; sh.red_f[1][warp] = mn; }
  __syncthreads();
  if (C > 1) cluster_wait();  // every rank runs: its shared memory may be written
  if (warp == 0) {
    mx = warp_max(sh.red_f[0][lane % SR_WARPS]);
    mn = -warp_max(-sh.red_f[1][lane % SR_WARPS]);
    if (lane < C) {
      peer(sh.mx, lane, C)[rank] = mx;
      peer(sh.mn, lane, C)[rank] = mn;
    }
  }
  cluster_barrier(C);
  mx = sh.mx[0];
  mn = sh.mn[0];
  for (int q = 1; q < C; q++) {
    mx = fmaxf(mx, sh.mx[q]);
    mn = fminf(mn, sh.mn[q]);
  }
  if (mx == -INFINITY) {  // nothing to draw from (the same for every rank)
    if (rank == 0 && tid == 0) {
      s.tokens[r] = -1;
      if (s.logprobs) s.logprobs[r] = -INFINITY;
    }
    return;
  }
  float4* mine = reinterpret_cast<float4*>(xs + tid * per);  // this thread's consecutive elements
  const int first_i = c0 - lead + tid * per;                 // index of the first (below 0 only in padding)
  if (mx == INFINITY) {  // the infinite ones share the mass: a row of 0 and -inf
    auto flat = [](float x) { return x == INFINITY ? 0.f : -INFINITY; };
    for (int i = 0; i < per / 4; i++) mine[i] = make_float4(flat(mine[i].x), flat(mine[i].y), flat(mine[i].z), flat(mine[i].w));
    mx = mn = 0.f;
    __syncthreads();
  }
  // ---- fp32 sum of the weights, first maximum, histogram of counts
  const float t1 = fminf(fmaxf(T > 0.f ? T : 1.f, 1e-30f), 1e30f);
  const float c2 = 1.4426950408889634f / t1;
  // log 2 of a weight: the product with 1 / (T ln 2) in two floats, so that its
  // rounding does not lean every weight the same way
  const float c2_lo = (float)(1.4426950408889634 / (double)t1 - (double)c2);
  const float deep = -200.f / c2;  // 2^-200 is 0 as well, and the products stay finite
  const float span = fminf(fmaxf(mx - mn, 1e-30f), SR_SPAN);
  const float bin_scale = (float)(SR_BINS - 1) / span;
  float u = s.u[r];
  if (!(u >= 0.f)) u = 0.f;
  const Row row{s, C, rank, r, per, first_i, slice, mx, span, bin_scale, t1, c2, c2_lo, deep, u,
                Weigh{(double)mx, -1.0 / (SR_STEP * (double)t1)}, k, top_p, (double)min_p, by_k, by_p, by_m};
  double own = 0;  // this thread's weights
  {
    // the maxima are counted, not summed: a row that is nearly certain keeps the
    // digits of what the other tokens share
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    unsigned ones = 0;
    int first = 0x7fffffff;
    if (need_bins) {
      row.each([&](const float (&x)[4], int) {
        float e[4];
        int b[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          e[j] = ex2f(row.octaves(x[j]));
          b[j] = row.bin_of(x[j]);
          if (e[j] < 1.f) part[j] += e[j];
          else ones++;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (b[j] < SR_BINS - 1) atomicAdd(&sh.hist[b[j]].x, 1u);  // the last bin is the rest
          if (e[j] > SR_HEAVY) atomicAdd(&sh.hist[b[j]].y, (unsigned)(__float_as_int(e[j] + 128.f) - 0x43000000));
        }
      });
    } else {
      row.each([&](const float (&x)[4], int i) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float e = ex2f(row.octaves(x[j]));
          if (e < 1.f) part[j] += e;
          else ones++;
          if (top1 && x[j] == mx) first = min(first, first_i + i + j);
        }
      });
    }
    double sum = ((double)part[0] + part[1]) + ((double)part[2] + part[3]);
    own = sum + ones;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    first = __reduce_min_sync(0xffffffffu, first);
    ones = __reduce_add_sync(0xffffffffu, ones);
    if (lane == 0) { sh.red_o[warp] = (u64)__double_as_longlong(sum); sh.red_c[warp] = (unsigned)first; sh.red_m[warp] = ones; }
    __syncthreads();
    if (warp == 0) {
      sum = __longlong_as_double((long long)sh.red_o[lane % SR_WARPS]);
#pragma unroll
      for (int d = SR_WARPS / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      first = __reduce_min_sync(0xffffffffu, (int)sh.red_c[lane % SR_WARPS]);
      ones = __reduce_add_sync(0xffffffffu, lane < SR_WARPS ? (unsigned)sh.red_m[lane] : 0u);
      if (lane < C) {
        peer(sh.sum, lane, C)[rank] = sum;
        peer(sh.ones, lane, C)[rank] = ones;
        peer(sh.first, lane, C)[rank] = first;
      }
    }
  }
  double pre = own;  // this thread's place in the slice's mass
  if (!top1 && !need_bins) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, pre, d);
      if (lane >= d) pre += v;
    }
    __syncthreads();  // red_m has been read
    if (lane == 31) sh.red_m[warp] = (u64)__double_as_longlong(pre);
    __syncthreads();
    pre -= own;
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++)
      if (w < warp) pre += __longlong_as_double((long long)sh.red_m[w]);
  }
  cluster_barrier(C);
  if (top1) {
    if (rank == 0 && tid == 0) {
      int f = 0x7fffffff;
      for (int q = 0; q < C; q++) f = min(f, sh.first[q]);
      row.finish(f, mx);
    }
    return;
  }

  if (!need_bins) {
    // ---- the whole row is kept: the element that the number falls into by the
    // fp32 weights is the right one where it lies further inside than these can
    // be off, the sum before it and its place in the sum both
    double z = 0, base = 0;
    for (int q = 0; q < C; q++) {
      if (q == rank) base = z;
      z += sh.sum[q] + sh.ones[q];
    }
    const double at = (double)u * z, margin = 2.0 * (double)row.off_by((float)z) * z;
    const double b = base + pre;
    const unsigned claim = __ballot_sync(0xffffffffu, at >= b && at < b + own);
    if (claim) {
      const int owner = __ffs(claim) - 1;
      double run = __shfl_sync(0xffffffffu, b, owner);
      const float* ox = xs + (warp * 32 + owner) * per;
      for (int i0 = 0; i0 < per; i0 += 32) {
        const int i = i0 + lane;
        const float x = i < per ? ox[i] : -INFINITY;
        const double e = ex2f(row.octaves(x));
        double upto = e;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += v;
        }
        upto += run;
        if (at - (upto - e) > margin && upto - at > margin) {
          row.finish(c0 - lead + (warp * 32 + owner) * per + i, x);
          for (int q = 0; q < C; q++) peer(&sh, q, C)->drawn = 1;
        }
        run = __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    cluster_barrier(C);
    if (sh.drawn) return;
  }

  int kbin = SR_BINS - 1, pbin = 0;
  unsigned kabove = 0;
  u64 all = 0;
  if (need_bins) {
    // ---- the first histogram over the cluster: a thread has SR_BPT neighbours.
    // Masses are a guess, checked below: sums of 2^-16 units where the bin's
    // weights are heavy, count * weight at the middle of the bin where they are light
    unsigned c1[SR_BPT] = {}, lower[SR_BPT] = {}, ct, c_in = 0;  // lower: of the ranks before this one
    u64 m1[SR_BPT] = {}, mt, m_in = 0;
#pragma unroll
    for (int q = 0; q < SR_MAX_CLUSTER; q++)
      if (q < C) {
        const uint4 v = *reinterpret_cast<const uint4*>(peer(sh.hist, q, C) + SR_BPT * tid);
        if (q == rank) {
          lower[0] = c1[0];
          lower[1] = c1[1];
        }
        c1[0] += v.x;
        m1[0] += v.y;
        c1[1] += v.z;
        m1[1] += v.w;
      }
#pragma unroll
    for (int b = 0; b < SR_BPT; b++) {
      const float mid = ex2f(-(float)(SR_BPT * tid + b) * (span / (float)(SR_BINS - 1)) * c2);
      m1[b] = mid > SR_HEAVY ? m1[b] << 16 : (u64)((float)c1[b] * mid * 4294967296.f);
      c_in += c1[b];
      m_in += m1[b];
    }
    block_scan(sh, m_in, c_in, &mt, &ct);
    c_in -= c1[0] + c1[1];  // what is above this thread's bins
    m_in -= m1[0] + m1[1];
    if (tid == 0) { sh.found[0] = sh.found[1] = SR_BINS - 1; sh.found_c = ct; sh.found_m = mt; }
    __syncthreads();
    if (by_k) {
      unsigned c = c_in;
      u64 m = m_in;
#pragma unroll
      for (int b = 0; b < SR_BPT; b++) {
        if (c < (unsigned)k && (unsigned)k <= c + c1[b]) {
          sh.found[0] = SR_BPT * tid + b;
          sh.found_c = c;
          sh.found_m = m + (u64)((float)m1[b] * ((float)(k - (int)c) / (float)c1[b]));
        }
        c += c1[b];
        m += m1[b];
      }
    }
    __syncthreads();
    kbin = sh.found[0];
    kabove = sh.found_c;
    if (by_p) {
      const u64 goal = max((u64)1, (u64)((double)sh.found_m * (double)top_p));
      u64 m = m_in;
#pragma unroll
      for (int b = 0; b < SR_BPT; b++) {
        if (m < goal && goal <= m + m1[b]) sh.found[1] = SR_BPT * tid + b;
        m += m1[b];
      }
      __syncthreads();
      pbin = min(kbin, sh.found[1]);
    }
    // ---- the bins that can be kept, and how many elements they hold
    int last = kbin;
    bool covers = by_k;  // the bins hold all that can stay, whatever the guess is worth
    if (!by_k) {
      if (by_p) last = min(SR_BINS - 1, pbin + 1);
      if (by_m) {  // min-p keeps max - x <= T ln(1 / min_p); two bins on the safe side
        const float reach = -log2f(min_p) / c2 * bin_scale;
        const int down = reach < (float)(SR_BINS - 4) ? (int)reach + 3 : SR_BINS - 1;
        covers = down <= last;
        last = min(last, down);
      }
    }
    __syncthreads();
    if (tid == last / SR_BPT) sh.found_c = last == SR_BINS - 1 ? (unsigned)s.V : c_in + c1[0] + (last % SR_BPT ? c1[1] : 0u);
    __syncthreads();
    if (sh.found_c <= SR_LIST) {
      // ---- candidates in index order, to rank 0: behind those of the ranks
      // before, whose number the histograms tell (the last bin is not counted
      // there, but rows so short have one rank)
      const float edge = 8388608.f + (float)last;
      auto candidate = [&](float x) { return row.bin_bits(x) <= edge && x > -INFINITY; };
      unsigned hits = 0, hits_t;
      u64 base = (SR_BPT * tid <= last ? lower[0] : 0) + (SR_BPT * tid + 1 <= last ? lower[1] : 0), base_t;
      u64 fours = 0;  // the groups of four that hold any: the bins fall with the logit, so the largest tells
      for (int i = 0; i < per / 4; i++) {
        const float4 v = mine[i];
        if (candidate(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)))) {
          fours |= 1ull << i;
          hits += candidate(v.x) + candidate(v.y) + candidate(v.z) + candidate(v.w);
        }
      }
      const unsigned own = hits;
      block_scan(sh, base, hits, &base_t, &hits_t);
      const int total = last == SR_BINS - 1 ? (int)hits_t : (int)sh.found_c;
      int2* to = peer(sh.list.xi, 0, C) + (int)base_t + hits - own;
      for (; fours; fours &= fours - 1) {
        const int i = __ffsll((long long)fours) - 1;
        const float4 v = mine[i];
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (candidate(x[j])) *to++ = make_int2(__float_as_int(x[j]), first_i + 4 * i + j);
      }
      cluster_barrier(C);
      const bool alone = !by_p || by_k;  // rank 0 needs nothing more of its peers
      if (alone && rank) return;
      // ---- rank 0 orders them: into their bins, whose beginnings the histogram
      // tells, then by counting inside a bin (a few elements; all of them when
      // they are equal). Thread t gets places each * t and on, with the exact mass before them
      u64 f[SR_EPT] = {}, o[SR_EPT] = {}, before[SR_EPT] = {};
      const int each_t = (total + SR_THREADS - 1) / SR_THREADS;
      if (rank == 0) {
        unsigned* begin = reinterpret_cast<unsigned*>(sh.hist);  // read last before the barrier above
        begin[SR_BPT * tid] = c_in;
        begin[SR_BPT * tid + 1] = c_in + c1[0];
        __syncthreads();
        for (int i = tid; i < total; i += SR_THREADS) {
          const float x = __int_as_float(sh.list.xi[i].x);
          sh.list.order[atomicAdd(&begin[row.bin_of(x)], 1u)] = ((u64)key_of(x) << 32) | (0xffffffffu - (unsigned)i);
        }
        __syncthreads();  // a bin begins where the one before it ended
        int at[SR_EPT];
#pragma unroll
        for (int j = 0; j < SR_EPT; j++) {
          const int e = tid + j * SR_THREADS;
          if (e >= total) continue;
          o[j] = sh.list.order[e];
          const int b = row.bin_of(of_key((uint32_t)(o[j] >> 32)));
          const int from = b ? (int)begin[b - 1] : 0, end = (int)begin[b];
          at[j] = from;
          for (int i = from; i < end; i++) at[j] += sh.list.order[i] > o[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SR_EPT; j++)
          if (tid + j * SR_THREADS < total) sh.list.order[at[j]] = o[j];
        __syncthreads();
        u64 m = 0, mt;
#pragma unroll
        for (int j = 0; j < SR_EPT; j++) {
          const int e = each_t * tid + j;
          o[j] = 0;
          if (j < each_t && e < total) {
            o[j] = sh.list.order[e];
            f[j] = row.weight(of_key((uint32_t)(o[j] >> 32)));
          }
          before[j] = m;
          m += f[j];
        }
        const u64 own_mass = m;
        unsigned zero = 0, zero_t;
        block_scan(sh, m, zero, &mt, &zero_t);
#pragma unroll
        for (int j = 0; j < SR_EPT; j++) before[j] += m - own_mass;
      }
      auto place = [&](int j) { return j < each_t ? min(each_t * tid + j, SR_LIST) : SR_LIST; };
      const int nk = by_k ? min(k, total) : total;
      for (int pass = 0;; pass++) {  // at most two: the second with the row's exact mass
        if (rank == 0) {
          u64 lo = 0, hi = 0;  // the running mass that top-p asks for, as far as it is known
          if (by_p) {
            if (by_k) {
              if (tid == 0) sh.found_m = 0;
              __syncthreads();
#pragma unroll
              for (int j = 0; j < SR_EPT; j++)
                if (place(j) == nk - 1) sh.found_m = before[j] + f[j];
              __syncthreads();
              lo = hi = row.share(sh.found_m);
            } else if (pass) {
              all = 0;
              for (int q = 0; q < C; q++) all += sh.all[q];
              lo = hi = row.share(all);
            } else {
              double z = 0;
              for (int q = 0; q < C; q++) z += sh.sum[q] + sh.ones[q];
              const double err = row.off_by((float)z);
              lo = row.share((u64)(z * (1.0 - err) * 35184372088832.0));  // 2^45
              hi = row.share((u64)(z * (1.0 + err) * 35184372088832.0) + 1);
            }
          }
          // kept masses in index order; two ends of the top-p mass must keep the same ones,
          // and a list that ends before them decides nothing
          bool unsure = false, past = false, ended = false;
          u64 kept[SR_EPT] = {};
#pragma unroll
          for (int j = 0; j < SR_EPT; j++) {
            if (place(j) < nk && (!by_p || before[j] < lo)) kept[j] = by_m || u == 0.f ? row.weight_kept(of_key((uint32_t)(o[j] >> 32))) : f[j];
            unsure |= by_p && place(j) < nk && before[j] >= lo && before[j] < hi;
            if (by_p && !covers && place(j) == total - 1) {
              ended = before[j] + f[j] < hi;
              past = before[j] + f[j] < lo;
            }
          }
          const int doubt = __syncthreads_or(unsure || ended), whole = __syncthreads_or(past);
          const int todo = whole ? SR_WHOLE : doubt ? SR_EXACT : SR_DONE;
          if (todo == SR_DONE) {
#pragma unroll
            for (int j = 0; j < SR_EPT; j++)
              if (place(j) < total) sh.list.order[0xffffffffu - (uint32_t)o[j]] = kept[j];
            __syncthreads();
            u64 m = 0, mass, fk[SR_EPT];
#pragma unroll
            for (int j = 0; j < SR_EPT; j++) {
              fk[j] = place(j) < total ? sh.list.order[place(j)] : 0;
              m += fk[j];
            }
            const u64 own_mass = m;
            unsigned zero = 0, zero_t;
            block_scan(sh, m, zero, &mass, &zero_t);
            const u64 to = row.draw(mass);
            u64 run = m - own_mass;
            int win = -1;
#pragma unroll
            for (int j = 0; j < SR_EPT; j++) {
              if (fk[j] && run < to && to <= run + fk[j]) win = place(j);
              run += fk[j];
            }
            if (win >= 0) row.finish(sh.list.xi[win].y, __int_as_float(sh.list.xi[win].x));
          } else if (tid < C) {
            peer(&sh, tid, C)->again = todo;
          }
        }
        if (alone) return;
        cluster_barrier(C);  // rank 0 has told its peers what it needs
        const int todo = sh.again;
        if (todo == SR_DONE) return;
        if (todo == SR_WHOLE) break;
        // the exact mass of the row
        all = 0;
        row.each([&](const float (&x)[4], int) {
#pragma unroll
          for (int j = 0; j < 4; j++) all += row.weight(x[j]);
        });
        all = warp_sum64(all);
        __syncthreads();  // `again` and red_m have been read
        if (lane == 0) sh.red_m[warp] = all;
        if (tid == 0) sh.again = SR_DONE;
        __syncthreads();
        if (warp == 0) {
          all = warp_sum64(lane < SR_WARPS ? sh.red_m[lane] : 0);
          if (lane == 0) peer(sh.all, 0, C)[rank] = all;
        }
        cluster_barrier(C);
      }
    }
  }

  const Row apart = row;  // in memory for this call only
  finish_long(apart, kbin, pbin, kabove);
}

std::mutex g_attr_mu;
bool g_attr_done[OPS_MAX_DEV];
int set_attributes(int device) {
  if (device < 0 || device >= OPS_MAX_DEV) {
    set_error("wg_sample_rows: device %d out of range", device);
    return WG_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lk(g_attr_mu);
  if (g_attr_done[device]) return WG_OK;
  WG_CHECK_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SR_SMEM_MAX));
  g_attr_done[device] = true;
  return WG_OK;
}

}  // namespace

int init_sample_rows(int device) { return set_attributes(device); }

int launch_sample_rows(const wg_sample& p, int device, cudaStream_t st) {
  WG_CHECK(set_attributes(device));
  // CTAs a row: 8 while they all fit the SMs, else 4 (two halves of a row of
  // 51866 fp32 leave one CTA to an SM), none with less than 2048 elements
  // (their exchanges cost more than such slices). Measured with 2 / 4 / 8 CTAs
  // at a top-k: one row of 51865 fp32 21 / 16 / 14 us, 48 of 51864 f16 22 / 21 /
  // 24, 320 of 51866 fp32 102 / 67 / 104.
  int C = p.R * 8 <= 148 ? 8 : 4;
  while (C > 1 && p.V <= 2048 * (C / 2)) C /= 2;
  // elements a thread: 4 times an odd number that covers the slice and its padding
  auto per_of = [&](int c) {
    const int each = (p.V + c - 1) / c + SR_PAD;
    return 4 * (((each + 4 * SR_THREADS - 1) / (4 * SR_THREADS)) | 1);
  };
  auto smem_of = [&](int c) { return SR_HEAD + (size_t)per_of(c) * SR_THREADS * 4; };
  while (C < SR_MAX_CLUSTER && smem_of(C) > SR_SMEM_MAX) C *= 2;
  const int per = per_of(C);
  const size_t smem = smem_of(C);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)p.R * C));
  cfg.blockDim = dim3(SR_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = C;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? at : at + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (C > 1 ? 1 : 0);
  return launch_check(cudaLaunchKernelEx(&cfg, sample_rows_kernel, p, C, per), "sample_rows");
}

}  // namespace wg

extern "C" int wg_sample_rows(const wg_sample* p, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_sample_rows";
  if (!p || p->R < 0 || p->R > (1 << 24) || p->V <= 0 || p->V > SR_MAX_V || p->ld < p->V) {
    set_error("%s: bad argument (V from 1 to %d, rows at least V apart)", what, SR_MAX_V);
    return WG_ERR_INVALID;
  }
  if (!dt_ok(p->dtype)) {
    set_error("%s: unsupported type %d", what, p->dtype);
    return WG_ERR_UNSUPPORTED;
  }
  if (p->R == 0) return WG_OK;
  if (!p->logits || !p->u || !p->tokens || reinterpret_cast<uintptr_t>(p->logits) % dt_bytes(p->dtype) ||
      !aligned4(p->u, p->temperature, p->top_k, p->top_p, p->min_p, p->tokens, p->logprobs)) {
    set_error("%s: null or misaligned tensor", what);
    return WG_ERR_INVALID;
  }
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  return launch_sample_rows(*p, device, reinterpret_cast<cudaStream_t>(stream));
}
