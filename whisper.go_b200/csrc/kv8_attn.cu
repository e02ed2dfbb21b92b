// kv8_attn.cu — attention over the 8-bit paged K/V cache (wg_kv8_attention).
//
// For query row i of a request of nq rows over len cached tokens
//   s_j = scale * sk_j * (q_i . k_j)     k_j, v_j: int8 codes, sk, sv: the page's scales
//   p_j = exp(s_j - max_j s_j)           over the visible j (causal: j <= len - nq + i)
//   o_i = (1 / sum_j p_j) * sum_j p_j * sv_j * v_j,   0 where nothing is visible
// in one pass over the cache with a running maximum and sum. At most 16 (query,
// grouped head) rows share a K/V head here; kv8_prompt.cu has the prompts.
//
// The codes are exact in f16, so both products run on mma.m16n8k16 (f16 in,
// fp32 accumulators); scales multiply the fp32 results. What bounds it is the
// cache's bytes (2 * D bytes per token and head), and next to them the
// instructions that turn a byte into an f16: 176 of the ~497 that a warp spends
// on 32 tokens of 64-wide heads. So:
//  - (query, grouped head) pairs that share a K/V head are one tile: single
//    tokens, beams and grouped heads take one read. Up to 8 of them are the
//    columns of the MMA and tokens (then dims) its 16 rows, which halves the
//    MMAs and accumulators; 9 to 16 are its rows;
//  - two bytes become 1152 + code by one byte permute, and codes by one packed
//    subtraction. (Left in and taken out through the accumulators the 1152 saves
//    that subtraction, 50.4 us against 51.8 in the cross case below, but 1152 *
//    sum q and 1152 * sum p leave their rounding behind: an output of small
//    values beside a strong zero was 10 % off.)
//  - what meets the codes in an MMA is f16 too: the softmax weights are lifted
//    and rounded (pack_weights), fp32 queries rounded to 11 bits (query_range)
//    as the f16 cache's cross-attention rounds them; their low parts would cost
//    as many MMAs again;
//  - every warp streams its own 32-token chunks through its own ring of
//    cp.async stages (no CTA barrier in the loop, no bounded wait needed: a
//    cp.async group always completes);
//  - the MMA's k order is free as long as both operands agree, so a thread
//    takes 16 consecutive codes of a token for Q.K^T (one 16-byte shared load
//    per 8 tokens) and 8 or 16 consecutive dims of 4 tokens for P.V;
//  - tokens are split over the CTAs of a cluster and joined through
//    distributed shared memory: one launch, no workspace in global memory.
// Measured: 64 utterances x 1500 tokens x 20 heads, 5 queries each (248 MB)
// 50 to 53 us = 4.7 to 4.95 TB/s, 71 to 75 % of the measured copy rate (issue
// slots 63 % busy);
// two requests of 60001 and ~29000 tokens, 8 heads of 128, 4 grouped queries
// (183 MB) 56 us = 3.3 TB/s (at most 16 CTAs a head: ~7 warps an SM, bound by
// each warp's own latency); 229 tokens of 6 heads 8 to 13 us a call, most of it
// the host's part and the launch.
#include <cooperative_groups.h>

#include <mutex>

#include "kv8_attn.cuh"

namespace wg {
namespace {

constexpr int AW = 4;        // warps per CTA (6 and 8 were slower at 128-wide heads: 52 -> 56, 67 us)
constexpr int CH = 32;       // tokens per chunk
constexpr int STAGES = 2;    // more hide no more: 3 and 4 stages left 64 x 1500 tokens at 52 us
template <int D>
constexpr int stage_bytes() { return 2 * CH * D + 32; }  // K, V, {sk[2], sv[2], page ok[2]}
template <int D>
constexpr int warp_bytes() { return STAGES * stage_bytes<D>(); }
template <int D>
constexpr int smem_bytes() { return AW * warp_bytes<D>(); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float column_max(float v) {  // over the lanes of one t
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
// Shared-memory byte offset of the 16-byte piece `part` of token tok in a
// [32][D] block. Swizzled so that a quarter-warp's 16-byte reads of K (two
// neighbouring tokens x 4 pieces) and a half-warp's 8-byte (D 64) or
// quarter-warp's 16-byte (D 128) reads of V (tokens 2t + i of t = 0..3) each
// touch every bank once.
template <int D>
__device__ __forceinline__ uint32_t k_off(int tok, int part) {
  if constexpr (D == 64) return tok * 64 + part * 16;
  return tok * 128 + ((part ^ ((tok & 1) << 2)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t v_off(int tok, int part) {
  if constexpr (D == 64) {  // 128-byte lines of two tokens
    const int line = tok >> 1, q = ((tok & 1) << 2) | part;
    return line * 128 + ((q ^ ((line & 3) << 1)) << 4);
  }
  return tok * 128 + ((part ^ (((tok >> 1) & 3) << 1)) << 4);
}

// A lane's share of 32 tokens of V: D/8 dims (from g) of tokens 2t, 2t + 1,
// 2t + 8 and 2t + 9 of either 16, offset by 128.
template <int D>
__device__ __forceinline__ void load_v(const uint8_t* vs, int g, int t, uint32_t (&w)[2][4][D / 32]) {
#pragma unroll
  for (int hf = 0; hf < 2; hf++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int tok = hf * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
      if constexpr (D == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(vs + v_off<D>(tok, g >> 1) + (g & 1) * 8);
        w[hf][i][0] = v.x ^ 0x80808080u;
        w[hf][i][1] = v.y ^ 0x80808080u;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(vs + v_off<D>(tok, g));
        w[hf][i][0] = v.x ^ 0x80808080u;
        w[hf][i][1] = v.y ^ 0x80808080u;
        w[hf][i][2] = v.z ^ 0x80808080u;
        w[hf][i][3] = v.w ^ 0x80808080u;
      }
    }
}

// HALF: at most 8 rows are live, so the MMA's rows 8..15 are not processed
// past the products. SMALL: 16-token pages (two pages, and scales, per chunk).
template <int D, bool HALF, bool SMALL>
__global__ void __launch_bounds__(AW * 32, D == 64 ? 5 : 2) decode_attn_kernel(const Kv8AttnArgs p) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();
  pdl_wait();
  constexpr int PARTS = D / 16;  // 16-byte pieces of a token
  constexpr int NT = D / 8;      // n-tiles of P.V
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const int h = unit / p.R, r = unit % p.R;
  const int page = 1 << p.shift;
  int q0 = __ldg(p.cu_q + r);
  int nq = __ldg(p.cu_q + r + 1) - q0;
  if (q0 < 0 || nq < 0 || q0 > p.n_q || nq > p.n_q - q0) nq = 0;
  const int rows = min(16, min(nq, p.max_q) * p.G);
  if (rows <= 0) return;  // the whole cluster: the request has no row
  const int len = min(max(__ldg(p.kv_lens + r), 0), (int)min((int64_t)p.max_pages << p.shift, (int64_t)0x7fffff00));
  const int* table = p.table + (int64_t)r * p.ldt;
  // tokens [0, lim) are visible to a row
  const int qa = g / p.G, qb = (g + 8) / p.G, qlast = (rows - 1) / p.G;
  const int lim_a = p.causal ? max(0, len - nq + qa + 1) : len;
  const int lim_b = p.causal ? max(0, len - nq + qb + 1) : len;
  const int hi = p.causal ? max(0, len - nq + qlast + 1) : len;
  const int lo_lim = p.causal ? max(0, len - nq + 1) : len;  // every row sees [0, lo_lim)
  const int nch = (hi + CH - 1) / CH, per = (nch + p.splits - 1) / p.splits;
  const int c_end = min(nch, (rank + 1) * per);
  int c = rank * per + warp;

  // ---- the warp's ring
  uint8_t* ring = smem + warp * warp_bytes<D>();
  const uint32_t ring_u = (uint32_t)__cvta_generic_to_shared(ring);
  const int pages = (len + page - 1) >> p.shift;
  auto page_id = [&](int chunk, int half) -> int {
    const int col = (chunk * CH + half * 16) >> p.shift;
    return chunk < c_end && col < pages ? __ldg(table + col) : -1;
  };
  // a lane's place in the first 512 bytes of a chunk's K and V, and in V's next
  // 512 (piece i is 512 i bytes further in memory; in the ring the swizzles
  // repeat every 512 bytes, V's of 128-wide heads every 1024)
  constexpr int PIECES = CH * D / 512;
  const uint32_t lane_k = k_off<D>(lane / PARTS, lane % PARTS), lane_v = CH * D + v_off<D>(lane / PARTS, lane % PARTS);
  const uint32_t lane_v1 = CH * D + v_off<D>(lane / PARTS + 32 / PARTS, lane % PARTS) - 512;
  const int64_t block = (int64_t)page * D, id_step = 2 * p.H * block, kv_step = p.H * block;
  const int8_t* lane_src = p.codes + h * block + lane * 16;
  const float* lane_scale = p.scales + h + (lane >> 1) * p.H;  // lanes 0..3: sk[0], sk[1], sv[0], sv[1]
  auto issue = [&](int chunk, uint32_t base, uint8_t* at, int id0, int id1) {
    const bool ok0 = (unsigned)id0 < (unsigned)p.num_pages, ok1 = SMALL ? (unsigned)id1 < (unsigned)p.num_pages : ok0;
    const int64_t page0 = (ok0 ? id0 : 0) * id_step, page1 = SMALL ? (ok1 ? id1 : 0) * id_step : 0;
    const int8_t* s0 = lane_src + page0 + (SMALL ? 0 : ((chunk * CH) & (page - 1)) * D);
    const int8_t* s1 = SMALL ? lane_src + page1 - 16 * D : s0;  // tokens 16..31 of 16-token pages
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const bool second = SMALL && i >= PIECES / 2;
      const int8_t* src = (second ? s1 : s0) + i * 512;
      cp16(base + lane_k + i * 512, src, second ? ok1 : ok0);
      cp16(base + ((i & 1) ? lane_v1 : lane_v) + i * 512, src + kv_step, second ? ok1 : ok0);
    }
    if (lane < 4) {
      const bool second = SMALL && (lane & 1);
      cp4(base + 2 * CH * D + lane * 4, lane_scale + (int64_t)(second ? (ok1 ? id1 : 0) : (ok0 ? id0 : 0)) * 2 * p.H,
          second ? ok1 : ok0);
    } else if (lane < 6) {
      reinterpret_cast<int*>(at + 2 * CH * D)[lane] = lane == 4 ? ok0 : ok1;
    }
  };
  int id0[STAGES], id1[STAGES];
#pragma unroll
  for (int s = 0; s < STAGES; s++) {
    id0[s] = page_id(c + s * AW, 0);
    id1[s] = SMALL ? page_id(c + s * AW, 1) : id0[s];
  }
#pragma unroll
  for (int s = 0; s < STAGES; s++) {
    if (c + s * AW < c_end)
      issue(c + s * AW, ring_u + s * stage_bytes<D>(), ring + s * stage_bytes<D>(), id0[s], id1[s]);
    cp_commit();
  }
  int nid0 = page_id(c + STAGES * AW, 0), nid1 = SMALL ? page_id(c + STAGES * AW, 1) : nid0;

  // ---- Q as A fragments: thread t of row g takes dims 16t..16t+15 of each
  // 64 (the 16 consecutive codes it reads of a token). Rows of bf16 or fp32
  // are scaled by a power of two so that they fit f16 (query_range).
  uint32_t qa_f[D / 16][4];
  float mul_a, mul_b;
  {
    float e[2];
    const float sign = p.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int half = 0; half < (HALF ? 1 : 2); half++) {
      const int row = g + half * 8;
      const bool live = row < rows;
      const int qi = row / p.G, hg = row % p.G;
      const int64_t base = (int64_t)(q0 + qi) * p.ldq + ((int64_t)h * p.G + hg) * D + 16 * t;
      float x[D / 4];
      float mx = 0.f;
      if (live && p.q_vec) {  // 16-bit types, 16-byte rows
#pragma unroll
        for (int i = 0; i < D / 4; i += 8) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + base + (i / 16) * 64 + i % 16));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 f = dt_unpack2(p.qdt, w[j]);
            x[i + 2 * j] = f.x;
            x[i + 2 * j + 1] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; i++) x[i] = live ? dt_load(p.q, base + (i / 16) * 64 + (i % 16), p.qdt) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 4; i++) mx = fmaxf(mx, fabsf(x[i]));
      mx = quad_max(mx);
      float up = sign;
      e[half] = 1.f;
      if (p.qdt != WG_DT_F16 && mx > 0.f && mx <= 3.402823466e38f) {
        query_range(mx, &up, &e[half]);
        up *= sign;
      }
#pragma unroll
      for (int j = 0; j < D / 16; j++) {  // MMA k step j: dims 16t + 4(j%4) .. +3 of 64-block j/4
        const int o = (j / 4) * 16 + (j % 4) * 4;
        qa_f[j][half] = pack_f16(x[o] * up, x[o + 1] * up);
        qa_f[j][2 + half] = pack_f16(x[o + 2] * up, x[o + 3] * up);
      }
    }
    mul_a = e[0] * fabsf(p.scale) * KV8_LOG2E;  // scores in units of log 2
    mul_b = HALF ? 0.f : e[1] * fabsf(p.scale) * KV8_LOG2E;
  }

  constexpr int OT = HALF ? D / 16 : NT;  // accumulator tiles
  float o_acc[OT][4];
#pragma unroll
  for (int j = 0; j < OT; j++) o_acc[j][0] = o_acc[j][1] = o_acc[j][2] = o_acc[j][3] = 0.f;
  // of rows g and g + 8, or with few rows of queries 2t and 2t + 1
  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
  float mul0 = 0.f, mul1 = 0.f;
  int lim0 = 0, lim1 = 0;
  if (HALF) {  // lane 4r + t holds row r's factors
    mul0 = __shfl_sync(0xffffffffu, mul_a, 8 * t);
    mul1 = __shfl_sync(0xffffffffu, mul_a, 8 * t + 4);
    lim0 = __shfl_sync(0xffffffffu, lim_a, 8 * t);
    lim1 = __shfl_sync(0xffffffffu, lim_a, 8 * t + 4);
  }

  for (int stage = 0; c < c_end; c += AW, stage = stage + 1 == STAGES ? 0 : stage + 1) {
    cp_wait<STAGES - 1>();
    __syncwarp();
    uint8_t* st = ring + stage * stage_bytes<D>();
    const float* sc = reinterpret_cast<const float*>(st + 2 * CH * D);
    const float sk0 = sc[0], sk1 = sc[1], sv0 = sc[2] * KV8_UNLIFT, sv1 = sc[3] * KV8_UNLIFT;
    const bool ok0 = reinterpret_cast<const int*>(sc)[4] != 0, ok1 = reinterpret_cast<const int*>(sc)[5] != 0;

    if constexpr (HALF) {
      // ---- at most 8 rows: tokens (then dims) are the MMA's 16 rows, queries
      // its 8 columns
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int b = 0; b < D / 64; b++) {
          const uint4 u4 = *reinterpret_cast<const uint4*>(st + k_off<D>(i * 16 + g, b * 4 + t));
          const uint4 v4 = *reinterpret_cast<const uint4*>(st + k_off<D>(i * 16 + 8 + g, b * 4 + t));
          const uint32_t u[4] = {u4.x ^ 0x80808080u, u4.y ^ 0x80808080u, u4.z ^ 0x80808080u, u4.w ^ 0x80808080u};
          const uint32_t v[4] = {v4.x ^ 0x80808080u, v4.y ^ 0x80808080u, v4.z ^ 0x80808080u, v4.w ^ 0x80808080u};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int ks = b * 4 + j;
            const uint32_t a0 = codes_f16<0x4140>(u[j]), a1 = codes_f16<0x4140>(v[j]);
            const uint32_t a2 = codes_f16<0x4342>(u[j]), a3 = codes_f16<0x4342>(v[j]);
            if (ks == 0) mma16816_zero(s[i], a0, a1, a2, a3, qa_f[0][0], qa_f[0][2]);
            else mma16816(s[i], a0, a1, a2, a3, qa_f[ks][0], qa_f[ks][2]);
          }
        }
        if (SMALL) {
#pragma unroll
          for (int x = 0; x < 4; x++) s[i][x] *= i ? sk1 : sk0;
        }
      }
      if ((c + 1) * CH > lo_lim || !ok0 || !ok1) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int j = c * CH + i * 16 + g;
          const bool ok = i ? ok1 : ok0;
          if (!ok || j >= lim0) s[i][0] = -INFINITY;
          if (!ok || j >= lim1) s[i][1] = -INFINITY;
          if (!ok || j + 8 >= lim0) s[i][2] = -INFINITY;
          if (!ok || j + 8 >= lim1) s[i][3] = -INFINITY;
        }
      }
      // running maximum; scores in units of log 2 are s * step (the sign of the
      // scale is in q; a step of 0, an all-zero page, is kept above 0 so that
      // masked scores stay -inf)
      const float step0 = fmaxf(SMALL ? mul0 : sk0 * mul0, 1e-37f), step1 = fmaxf(SMALL ? mul1 : sk0 * mul1, 1e-37f);
      float x0 = column_max(fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])));
      float x1 = column_max(fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3])));
      x0 = fmaxf(m_a, x0 * step0);
      x1 = fmaxf(m_b, x1 * step1);
      const float ref0 = x0 == -INFINITY ? 0.f : x0, ref1 = x1 == -INFINITY ? 0.f : x1;
      if (__any_sync(0xffffffffu, x0 != m_a || x1 != m_b)) {
        const float al0 = ex2(m_a - ref0), al1 = ex2(m_b - ref1);
        l_a *= al0;
        l_b *= al1;
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          o_acc[j][0] *= al0;
          o_acc[j][1] *= al1;
          o_acc[j][2] *= al0;
          o_acc[j][3] *= al1;
        }
        m_a = x0;
        m_b = x1;
      }
      // lifted weights rounded to f16, queries in rows: the other operand of P.V.
      // The products are rounded as the maximum's was: fused with the sum, a
      // maximum of 2^25 and more would miss itself by octaves
      const float lift0 = KV8_LIFT - ref0, lift1 = KV8_LIFT - ref1;
      uint32_t pb[2][2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        pb[i][0] = transpose8(pack_weights(ex2(__fmul_rn(s[i][0], step0) + lift0), ex2(__fmul_rn(s[i][1], step1) + lift1)));
        pb[i][1] = transpose8(pack_weights(ex2(__fmul_rn(s[i][2], step0) + lift0), ex2(__fmul_rn(s[i][3], step1) + lift1)));
      }
      // their sums, by the same MMA over a matrix of ones, go into l (so that the
      // rounded weights sum to one)
      constexpr uint32_t ONES = 0x3c003c00u;
      float rs[2][4];
      mma16816_zero(rs[0], ONES, ONES, ONES, ONES, pb[0][0], pb[0][1]);
      if (SMALL) mma16816_zero(rs[1], ONES, ONES, ONES, ONES, pb[1][0], pb[1][1]);
      else mma16816(rs[0], ONES, ONES, ONES, ONES, pb[1][0], pb[1][1]);
      l_a = fmaf(SMALL ? rs[0][0] + rs[1][0] : rs[0][0], KV8_UNLIFT, l_a);
      l_b = fmaf(SMALL ? rs[0][1] + rs[1][1] : rs[0][1], KV8_UNLIFT, l_b);
      // ---- V^T.P^T: rows g and g + 8 of m-tile j are dims 2j and 2j + 1 of lane g's D/8
      const uint8_t* vs = st + CH * D;
      constexpr int VW = D / 32;  // words of a lane's dims per token
      uint32_t w[2][4][VW];
      load_v<D>(vs, g, t, w);
#pragma unroll
      for (int k = 0; k < VW; k++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {  // dims 4k + 2e and 4k + 2e + 1
          const int j = 2 * k + e;
          float acc[2][4];
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            const uint32_t z0 = __byte_perm(w[hf][0][k], w[hf][1][k], e ? 0x7362 : 0x5140);
            const uint32_t z1 = __byte_perm(w[hf][2][k], w[hf][3][k], e ? 0x7362 : 0x5140);
            const uint32_t a0 = codes_f16<0x4140>(z0), a1 = codes_f16<0x4342>(z0);
            const uint32_t a2 = codes_f16<0x4140>(z1), a3 = codes_f16<0x4342>(z1);
            if (SMALL || hf == 0) mma16816_zero(acc[hf], a0, a1, a2, a3, pb[hf][0], pb[hf][1]);
            else mma16816(acc[0], a0, a1, a2, a3, pb[1][0], pb[1][1]);
          }
#pragma unroll
          for (int x = 0; x < 4; x++) {
            o_acc[j][x] = fmaf(sv0, acc[0][x], o_acc[j][x]);
            if (SMALL) o_acc[j][x] = fmaf(sv1, acc[1][x], o_acc[j][x]);
          }
        }
      }
    } else {
      // ---- q . codes of 4 n-tiles of 8 tokens, in units of the page's step
      // (both pages' steps brought to one where they differ)
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; n++) {
#pragma unroll
        for (int b = 0; b < D / 64; b++) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(st + k_off<D>(n * 8 + g, b * 4 + t));
          const uint32_t w[4] = {w4.x ^ 0x80808080u, w4.y ^ 0x80808080u, w4.z ^ 0x80808080u, w4.w ^ 0x80808080u};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (b == 0 && j == 0)
              mma16816_zero(s[n], qa_f[0], codes_f16<0x4140>(w[0]), codes_f16<0x4342>(w[0]));
            else
              mma16816(s[n], qa_f[b * 4 + j], codes_f16<0x4140>(w[j]), codes_f16<0x4342>(w[j]));
          }
        }
        if (SMALL && n >= 2) {
#pragma unroll
          for (int x = 0; x < 4; x++) s[n][x] *= sk1;
        } else if (SMALL) {
#pragma unroll
          for (int x = 0; x < 4; x++) s[n][x] *= sk0;
        }
      }
      if ((c + 1) * CH > lo_lim || !ok0 || !ok1) {
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const int j = c * CH + n * 8 + 2 * t;
          const bool ok = n < 2 ? ok0 : ok1;
          if (!ok || j >= lim_a) s[n][0] = -INFINITY;
          if (!ok || j + 1 >= lim_a) s[n][1] = -INFINITY;
          if (!ok || j >= lim_b) s[n][2] = -INFINITY;
          if (!ok || j + 1 >= lim_b) s[n][3] = -INFINITY;
        }
      }
      // ---- running maximum; scores in units of log 2 are s * step (the sign of
      // the scale is in q; a step of 0, an all-zero page, is kept above 0 so that
      // masked scores stay -inf)
      const float step_a = fmaxf(SMALL ? mul_a : sk0 * mul_a, 1e-37f), step_b = fmaxf(SMALL ? mul_b : sk0 * mul_b, 1e-37f);
      float x_a = fmaxf(s[0][0], s[0][1]), x_b = fmaxf(s[0][2], s[0][3]);
#pragma unroll
      for (int n = 1; n < 4; n++) {
        x_a = fmaxf(x_a, fmaxf(s[n][0], s[n][1]));
        x_b = fmaxf(x_b, fmaxf(s[n][2], s[n][3]));
      }
      // an empty chunk stays -inf (0 * -inf would not)
      x_a = quad_max(x_a);
      x_a = x_a == -INFINITY ? m_a : fmaxf(m_a, x_a * step_a);
      x_b = quad_max(x_b);
      x_b = x_b == -INFINITY ? m_b : fmaxf(m_b, x_b * step_b);
      const float ref_a = x_a == -INFINITY ? 0.f : x_a, ref_b = x_b == -INFINITY ? 0.f : x_b;
      const bool moved = x_a != m_a || x_b != m_b;
      if (__any_sync(0xffffffffu, moved)) {
        const float al_a = ex2(m_a - ref_a), al_b = ex2(m_b - ref_b);
        l_a *= al_a;
        l_b *= al_b;
#pragma unroll
        for (int j = 0; j < NT; j++) {
          o_acc[j][0] *= al_a;
          o_acc[j][1] *= al_a;
          o_acc[j][2] *= al_b;
          o_acc[j][3] *= al_b;
        }
        m_a = x_a;
        m_b = x_b;
      }
      // lifted weights rounded to f16 for the MMA (products rounded as the maximum's)
      const float lift_a = KV8_LIFT - ref_a, lift_b = KV8_LIFT - ref_b;
      uint32_t pf[2][4];
#pragma unroll
      for (int n = 0; n < 4; n++) {
        pf[n >> 1][(n & 1) * 2] = pack_weights(ex2(__fmul_rn(s[n][0], step_a) + lift_a), ex2(__fmul_rn(s[n][1], step_a) + lift_a));
        pf[n >> 1][(n & 1) * 2 + 1] =
            pack_weights(ex2(__fmul_rn(s[n][2], step_b) + lift_b), ex2(__fmul_rn(s[n][3], step_b) + lift_b));
      }
      // their row sums, by the same MMA over a matrix of ones, go into l (so that
      // the rounded weights sum to one)
      float rs[2][4];
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        if (hf == 1 && !SMALL) mma16816(rs[0], pf[1], 0x3c003c00u, 0x3c003c00u);
        else mma16816_zero(rs[hf], pf[hf], 0x3c003c00u, 0x3c003c00u);
      }
      l_a = fmaf(SMALL ? rs[0][0] + rs[1][0] : rs[0][0], KV8_UNLIFT, l_a);
      l_b = fmaf(SMALL ? rs[0][2] + rs[1][2] : rs[0][2], KV8_UNLIFT, l_b);
      // ---- P.V: n-tile j of lane g is dim g * (D/8) + j; tokens 2t, 2t+1, 2t+8, 2t+9 of each 16
      const uint8_t* vs = st + CH * D;
      constexpr int VW = D / 32;  // words of a lane's dims per token
      uint32_t w[2][4][VW];
      load_v<D>(vs, g, t, w);
#pragma unroll
      for (int k = 0; k < VW; k++) {
        uint32_t z[2][4];  // bytes (token 0, token 1) of dims 0,1 | 2,3; the same of tokens 2, 3
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          z[hf][0] = __byte_perm(w[hf][0][k], w[hf][1][k], 0x5140);
          z[hf][1] = __byte_perm(w[hf][0][k], w[hf][1][k], 0x7362);
          z[hf][2] = __byte_perm(w[hf][2][k], w[hf][3][k], 0x5140);
          z[hf][3] = __byte_perm(w[hf][2][k], w[hf][3][k], 0x7362);
        }
#pragma unroll
        for (int dd = 0; dd < 4; dd++) {
          const int j = k * 4 + dd;
          float acc[2][4];
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            const uint32_t b0 = (dd & 1) ? codes_f16<0x4342>(z[hf][dd >> 1]) : codes_f16<0x4140>(z[hf][dd >> 1]);
            const uint32_t b1 = (dd & 1) ? codes_f16<0x4342>(z[hf][2 + (dd >> 1)]) : codes_f16<0x4140>(z[hf][2 + (dd >> 1)]);
            if (SMALL || hf == 0) mma16816_zero(acc[hf], pf[hf], b0, b1);
            else mma16816(acc[0], pf[1], b0, b1);
          }
#pragma unroll
          for (int x = 0; x < 4; x++) {
            o_acc[j][x] = fmaf(sv0, acc[0][x], o_acc[j][x]);
            if (SMALL) o_acc[j][x] = fmaf(sv1, acc[1][x], o_acc[j][x]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (c + STAGES * AW < c_end) issue(c + STAGES * AW, ring_u + stage * stage_bytes<D>(), st, nid0, nid1);
    cp_commit();
    nid0 = page_id(c + (STAGES + 1) * AW, 0);
    nid1 = SMALL ? page_id(c + (STAGES + 1) * AW, 1) : nid0;
  }
  cp_wait<0>();

  // ---- join the warps: (m, l, O) of each in its own ring's memory
  __syncwarp();
  float* wo = reinterpret_cast<float*>(ring);  // [16][D] O, then [16] m, [16] l
  {
    if constexpr (HALF) {
      // lane (g, t) holds dims g * D/8 .. of queries 2t and 2t + 1
#pragma unroll
      for (int cc = 0; cc < 2; cc++)
#pragma unroll
        for (int j = 0; j < D / 16; j += 2)
          *reinterpret_cast<float4*>(wo + (2 * t + cc) * D + g * NT + 2 * j) =
              make_float4(o_acc[j][cc], o_acc[j][2 + cc], o_acc[j + 1][cc], o_acc[j + 1][2 + cc]);
      if (g == 0) {
        wo[16 * D + 2 * t] = m_a;
        wo[16 * D + 2 * t + 1] = m_b;
        wo[16 * D + 16 + 2 * t] = l_a;
        wo[16 * D + 17 + 2 * t] = l_b;
      }
    } else {
      // lane (g, t) holds dims 2t * D/8 .. (2t + 2) * D/8 - 1 of rows g, g + 8
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int cc = 0; cc < 2; cc++)
#pragma unroll
          for (int j = 0; j < NT; j += 4)
            *reinterpret_cast<float4*>(wo + (g + half * 8) * D + (2 * t + cc) * NT + j) =
                make_float4(o_acc[j][half * 2 + cc], o_acc[j + 1][half * 2 + cc], o_acc[j + 2][half * 2 + cc],
                            o_acc[j + 3][half * 2 + cc]);
      if (t == 0) {
        wo[16 * D + g] = m_a;
        wo[16 * D + 16 + g] = l_a;
        wo[16 * D + g + 8] = m_b;
        wo[16 * D + 24 + g] = l_b;
      }
    }
  }
  __syncthreads();
  // CTA total into warp 0's block: each (row, 4 dims) by one thread
  constexpr int WF = warp_bytes<D>() / 4;  // floats between the warps' blocks
  float* cta = reinterpret_cast<float*>(smem);
  float* cta_ml = cta + AW * WF;  // [16] m, [16] l of the CTA, past every ring
  for (int row = tid; row < rows; row += AW * 32) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < AW; k++) m = fmaxf(m, cta[k * WF + 16 * D + row]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < AW; k++) l += cta[k * WF + 16 * D + 16 + row] * ex2(cta[k * WF + 16 * D + row] - ref);
    cta_ml[row] = m;
    cta_ml[16 + row] = l;
  }
  for (int i = tid; i < rows * (D / 4); i += AW * 32) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < AW; k++) m = fmaxf(m, cta[k * WF + 16 * D + row]);
    const float ref = m == -INFINITY ? 0.f : m;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < AW; k++) {
      const float f = ex2(cta[k * WF + 16 * D + row] - ref);
      const float4 v = *reinterpret_cast<const float4*>(cta + k * WF + row * D + d);
      a.x = fmaf(v.x, f, a.x);
      a.y = fmaf(v.y, f, a.y);
      a.z = fmaf(v.z, f, a.z);
      a.w = fmaf(v.w, f, a.w);
    }
    // in place: this thread alone reads and writes these four floats of every warp's block
    *reinterpret_cast<float4*>(cta + row * D + d) = a;
  }
  // ---- join the cluster's CTAs: rank k finishes every splits-th (row, 4 dims)
  namespace cg = cooperative_groups;
  if (p.splits > 1) cg::this_cluster().sync();
  else __syncthreads();
  for (int i = tid * p.splits + rank; i < rows * (D / 4); i += AW * 32 * p.splits) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.splits; k++) {
      const float* peer = p.splits > 1 ? cg::this_cluster().map_shared_rank(cta, k) : cta;
      const float pm = peer[AW * WF + row], pl = peer[AW * WF + 16 + row];
      const float4 v = *reinterpret_cast<const float4*>(peer + row * D + d);
      const float nm = fmaxf(m, pm), ref = nm == -INFINITY ? 0.f : nm;
      const float fo = ex2(m - ref), fn = ex2(pm - ref);
      l = l * fo + pl * fn;
      a.x = a.x * fo + v.x * fn;
      a.y = a.y * fo + v.y * fn;
      a.z = a.z * fo + v.z * fn;
      a.w = a.w * fo + v.w * fn;
      m = nm;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // nothing visible: zeros; NaN stays
    const int qi = row / p.G, hg = row % p.G;
    const int64_t at = (int64_t)(q0 + qi) * p.ldo + ((int64_t)h * p.G + hg) * D + d;
    if (p.o_vec) {
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) =
          make_uint2(dt_pack2(p.odt, a.x * inv, a.y * inv), dt_pack2(p.odt, a.z * inv, a.w * inv));
    } else {
      dt_store(p.out, at, p.odt, a.x * inv);
      dt_store(p.out, at + 1, p.odt, a.y * inv);
      dt_store(p.out, at + 2, p.odt, a.z * inv);
      dt_store(p.out, at + 3, p.odt, a.w * inv);
    }
  }
  if (p.splits > 1) cg::this_cluster().sync();  // peers may still be reading this CTA
}

typedef void (*AttnKernel)(const Kv8AttnArgs);
template <int D>
AttnKernel pick(bool half, bool small) {
  if (half) return small ? decode_attn_kernel<D, true, true> : decode_attn_kernel<D, true, false>;
  return small ? decode_attn_kernel<D, false, true> : decode_attn_kernel<D, false, false>;
}

std::mutex g_attr_mu;
bool g_attr_done[OPS_MAX_DEV];

int set_attributes(int device) {
  if (device >= OPS_MAX_DEV) {
    set_error("wg_kv8_attention: device %d out of range", device);
    return WG_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lk(g_attr_mu);
  if (g_attr_done[device]) return WG_OK;
  for (int i = 0; i < 4; i++) {
    AttnKernel k64 = pick<64>(i & 1, i & 2), k128 = pick<128>(i & 1, i & 2);
    WG_CHECK_CUDA(cudaFuncSetAttribute(k64, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<64>() + 128));
    WG_CHECK_CUDA(cudaFuncSetAttribute(k128, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<128>() + 128));
    WG_CHECK_CUDA(cudaFuncSetAttribute(k64, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    WG_CHECK_CUDA(cudaFuncSetAttribute(k128, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  }
  WG_CHECK(kv8_prompt_attributes());
  g_attr_done[device] = true;
  return WG_OK;
}

}  // namespace

int init_kv8_attention(int device) { return set_attributes(device); }

// The launch behind wg_kv8_attention (arguments checked, device current).
int launch_kv8_attention(const wg_kv8& c, const wg_kv8_attn& p, int device, cudaStream_t st) {
  WG_CHECK(set_attributes(device));
  const int G = p.n_head / c.n_kv_head;
  const int max_q = p.max_q < p.n_q ? p.max_q : p.n_q;  // no request has more: a loose bound makes no empty tiles
  Kv8AttnArgs a{};
  a.codes = c.codes; a.scales = c.scales; a.num_pages = c.num_pages; a.shift = log2_of(c.page);
  a.H = c.n_kv_head; a.G = G; a.q = p.q; a.ldq = p.ldq; a.qdt = p.q_dtype; a.cu_q = p.cu_q; a.n_q = p.n_q;
  a.kv_lens = p.kv_lens; a.table = p.block_table; a.ldt = p.ld_table; a.max_pages = p.max_pages; a.R = p.n_requests;
  a.causal = p.causal; a.max_q = max_q; a.scale = p.scale; a.out = p.out; a.ldo = p.ldo; a.odt = p.out_dtype;
  a.q_vec = p.q_dtype != WG_DT_F32 && aligned16(p.q) && p.ldq % 8 == 0;
  a.o_vec = aligned16(p.out) && p.ldo % 8 == 0;
  const int64_t rows = (int64_t)max_q * G;
  const int64_t kv = p.max_kv < ((int64_t)p.max_pages << a.shift) ? p.max_kv : (int64_t)p.max_pages << a.shift;
  if (rows > 16) return launch_kv8_prompt(a, c.head_dim, kv, st);  // more than one MMA's rows
  const int64_t units = (int64_t)c.n_kv_head * p.n_requests;
  const int64_t chunks = (kv + CH - 1) / CH;
  // CTAs per (request, K/V head): enough for two rounds of the SMs' resident CTAs, no less
  // than two chunks for each warp, and no CTA with more than 64 chunks
  // (2048 tokens), so that one long request among short ones is spread too
  int64_t s = (148 * 6 + units - 1) / units;
  if (s > chunks / (2 * AW)) s = chunks / (2 * AW);
  if (s < (chunks + 63) / 64) s = (chunks + 63) / 64;
  a.splits = (int)(s < 1 ? 1 : s > KV8_MAX_SPLIT ? KV8_MAX_SPLIT : s);
  if (units * a.splits > 0x7fffffffLL) {
    set_error("wg_kv8_attention: %lld CTAs are more than a grid holds", (long long)(units * a.splits));
    return WG_ERR_INVALID;
  }
  const bool d64 = c.head_dim == 64;
  AttnKernel k = d64 ? pick<64>(rows <= 8, c.page == 16) : pick<128>(rows <= 8, c.page == 16);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * a.splits));
  cfg.blockDim = dim3(AW * 32);
  cfg.dynamicSmemBytes = (d64 ? smem_bytes<64>() : smem_bytes<128>()) + 128;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.splits;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? at : at + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (a.splits > 1 ? 1 : 0);
  return launch_check(cudaLaunchKernelEx(&cfg, k, a), "kv8_attention");
}

}  // namespace wg

extern "C" int wg_kv8_attention(const wg_kv8* cache, const wg_kv8_attn* p, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_kv8_attention";
  WG_CHECK(kv8_check(what, cache));
  if (!p || p->n_requests < 0 || p->n_q < 0 || p->max_q < 0 || p->max_kv < 0 || p->max_pages < 0 ||
      p->ld_table < p->max_pages) {
    set_error("%s: bad argument", what);
    return WG_ERR_INVALID;
  }
  if (p->n_head <= 0 || p->n_head % cache->n_kv_head) {
    set_error("%s: %d query heads over %d K/V heads", what, p->n_head, cache->n_kv_head);
    return WG_ERR_INVALID;
  }
  if (!dt_ok(p->q_dtype) || (p->out_dtype != WG_DT_F16 && p->out_dtype != WG_DT_BF16)) {
    set_error("%s: unsupported types (q %d, out %d: out is f16 or bf16)", what, p->q_dtype, p->out_dtype);
    return WG_ERR_UNSUPPORTED;
  }
  if (!(p->scale == p->scale) || p->scale > 3.4e38f || p->scale < -3.4e38f) {
    set_error("%s: the scale is not finite", what);
    return WG_ERR_INVALID;
  }
  if (p->n_requests == 0 || p->n_q == 0 || p->max_q == 0) return WG_OK;
  // the kernels count a head's (query, grouped head) rows, rounded up to a tile, in 32 bits
  if ((int64_t)(p->max_q < p->n_q ? p->max_q : p->n_q) * (p->n_head / cache->n_kv_head) > KV8_MAX_ATTN_ROWS) {
    set_error("%s: %d query rows of %d grouped heads are too many", what, p->n_q, p->n_head / cache->n_kv_head);
    return WG_ERR_INVALID;
  }
  const int64_t width = (int64_t)p->n_head * cache->head_dim;
  if (!p->q || !p->out || !p->cu_q || !p->kv_lens || (p->max_pages > 0 && !p->block_table) || p->ldq < width ||
      p->ldo < width || reinterpret_cast<uintptr_t>(p->q) % dt_bytes(p->q_dtype) ||
      reinterpret_cast<uintptr_t>(p->out) % 2 || !aligned4(p->cu_q, p->kv_lens, p->block_table)) {
    set_error("%s: null or misaligned tensor, or rows closer than %lld elements", what, (long long)width);
    return WG_ERR_INVALID;
  }
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  return launch_kv8_attention(*cache, *p, device, reinterpret_cast<cudaStream_t>(stream));
}
