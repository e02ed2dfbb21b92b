// kv8_prompt.cu — attention of prompts over the 8-bit paged K/V cache: more
// than 16 (query, grouped head) rows share a K/V head (wg_kv8_attention).
//
// The mathematics is kv8_attn.cu's. With many rows the conversion of codes to
// f16 is the work that repeats, so a CTA of 4 warps takes 64 rows and converts
// every 64-token chunk once for all of them: codes come from memory into
// registers one chunk ahead, go as f16 into a double-buffered shared tile, and
// each warp runs its 16 rows on mma.m16n8k16 with ldmatrix. Chunks past the
// last visible token of the tile are never read. Few tiles over many tokens
// are split over a cluster and joined through distributed shared memory.
//
// The bound would be the MMA (one m16n8k16 per ~9 cycles and SM quarter,
// measured) and the shared-memory reads that feed it (32 ldmatrix.x4 for 64
// MMAs per chunk and warp at 64-wide heads). At prompts of a text context it is
// latency: a tile has 1 to 7 chunks, and as much again goes into its start (the
// request, its pages, the codes, Q) and its end. Measured: 16 ragged prompts of
// up to 448 tokens, 20 heads, bf16: 37.5 us (61 us on 16-row tiles), 83 TFLOP/s
// with the tensor pipe 24 % busy; 4 CTAs an SM against 3: 38 / 42 us.
#include <cooperative_groups.h>

#include "kv8_attn.cuh"

namespace wg {
namespace {

namespace cg = cooperative_groups;

constexpr int PW = 4;        // warps
constexpr int PR = PW * 16;  // rows of a tile
constexpr int PT = 64;       // tokens of a chunk

// Byte offset of the 16-byte piece c of token tok in a [PT][D] f16 tile:
// eight tokens' pieces of one c fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t f_off(int tok, int c) { return tok * D * 2 + ((c ^ (tok & 7)) << 4); }

template <int D>
constexpr int tile_bytes() { return PT * D * 2; }
// two buffers of K and V, then per buffer and 16 tokens {sk, sv, page ok, -}
template <int D>
constexpr int prompt_smem() { return 4 * tile_bytes<D>() + 2 * 4 * 16; }
static_assert(PR * 64 * 4 + PR * 8 <= 4 * PT * 64 * 2 && PR * 128 * 4 + PR * 8 <= 4 * PT * 128 * 2,
              "the join's sums fit the tiles' memory");

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

// GT: tokens of a chunk that share a page, and so scales (16, 32 or 64)
template <int D, int GT>
__global__ void __launch_bounds__(PW * 32, D == 64 ? 4 : 2) prompt_attn_kernel(const Kv8AttnArgs p) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();
  pdl_wait();
  constexpr int PARTS = D / 16;                  // 16-byte pieces of a token's codes
  constexpr int NP = PT * PARTS / (PW * 32);     // pieces of K (and of V) a thread converts
  constexpr int NT = D / 8, KS = D / 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  // the last rows of a causal prompt see the most tokens: their tiles start first
  const int tile = p.tiles - 1 - unit / (p.H * p.R), h = unit % p.H, r = unit / p.H % p.R;
  const int page = 1 << p.shift;
  int q0 = __ldg(p.cu_q + r);
  int nq = __ldg(p.cu_q + r + 1) - q0;
  if (q0 < 0 || nq < 0 || q0 > p.n_q || nq > p.n_q - q0) nq = 0;
  const int row0 = tile * PR;
  const int rows = min(PR, min(nq, p.max_q) * p.G - row0);
  if (rows <= 0) return;  // the whole cluster: no row of this tile exists
  const int len = min(max(__ldg(p.kv_lens + r), 0), (int)min((int64_t)p.max_pages << p.shift, (int64_t)0x7fffff00));
  const int* table = p.table + (int64_t)r * p.ldt;
  const int ra = warp * 16 + g, rb = ra + 8;  // this thread's rows of the tile
  // tokens [0, lim) are visible to a row
  const int lim_a = p.causal ? max(0, len - nq + (row0 + ra) / p.G + 1) : len;
  const int lim_b = p.causal ? max(0, len - nq + (row0 + rb) / p.G + 1) : len;
  const int hi = p.causal ? max(0, len - nq + (row0 + rows - 1) / p.G + 1) : len;
  const int warp_lo = p.causal ? max(0, len - nq + (row0 + warp * 16) / p.G + 1) : len;  // all rows of the warp see it
  const int nch = (hi + PT - 1) / PT, per = (nch + p.splits - 1) / p.splits;
  const int c_end = min(nch, (rank + 1) * per);
  int c = rank * per;

  // ---- codes of a chunk: from memory into registers, then as f16 into a buffer
  const int pages = (len + page - 1) >> p.shift;
  uint4 kraw[NP], vraw[NP];
  float sk = 0.f, sv = 0.f;  // threads 0..3: scales of 16 tokens
  int ok = 0;
  auto id_of = [&](int token) {
    const int col = token >> p.shift, id = col < pages ? __ldg(table + col) : -1;
    return (unsigned)id < (unsigned)p.num_pages ? id : -1;
  };
  const int64_t kv_step = (int64_t)p.H * page * D;
  auto fetch = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int idx = i * PW * 32 + tid, tok = chunk * PT + idx / PARTS, part = idx % PARTS;
      const int id = id_of(tok);
      kraw[i] = vraw[i] = make_uint4(0, 0, 0, 0);
      if (id >= 0) {
        const int8_t* src = p.codes + (((int64_t)id * 2 * p.H + h) * page + (tok & (page - 1))) * D + part * 16;
        kraw[i] = __ldg(reinterpret_cast<const uint4*>(src));
        vraw[i] = __ldg(reinterpret_cast<const uint4*>(src + kv_step));
      }
    }
    if (tid < 4) {
      const int id = id_of(chunk * PT + tid * 16);
      ok = id >= 0;
      const float* s = p.scales + (int64_t)max(id, 0) * 2 * p.H + h;
      sk = ok ? __ldg(s) : 0.f;
      sv = ok ? __ldg(s + p.H) : 0.f;
    }
  };
  auto convert = [&](uint8_t* to, const uint4 (&raw)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int idx = i * PW * 32 + tid, tok = idx / PARTS, part = idx % PARTS;
      const uint32_t w[4] = {raw[i].x ^ 0x80808080u, raw[i].y ^ 0x80808080u, raw[i].z ^ 0x80808080u, raw[i].w ^ 0x80808080u};
#pragma unroll
      for (int k = 0; k < 2; k++)
        *reinterpret_cast<uint4*>(to + f_off<D>(tok, part * 2 + k)) =
            make_uint4(codes_f16<0x4140>(w[2 * k]), codes_f16<0x4342>(w[2 * k]), codes_f16<0x4140>(w[2 * k + 1]),
                       codes_f16<0x4342>(w[2 * k + 1]));
    }
  };
  auto meta = [&](int buf) { return reinterpret_cast<float4*>(smem + 4 * tile_bytes<D>()) + buf * 4; };
  if (c < c_end) fetch(c);

  // ---- Q through the second buffer: rows of bf16 or fp32 are scaled by a power
  // of two to fit f16 (query_range); D/8 lanes take a row, 8 dims each
  uint32_t qf[KS][4];
  float mul[2];
  {
    const float sign = p.scale < 0.f ? -1.f : 1.f;
    uint8_t* qs = smem + 2 * tile_bytes<D>();
    float* row_mul = reinterpret_cast<float*>(smem + 3 * tile_bytes<D>());
    constexpr int RL = D / 8;  // lanes of a row
#pragma unroll
    for (int i = 0; i < PR * RL / (PW * 32); i++) {
      const int idx = i * PW * 32 + tid, row = idx / RL, c8 = idx % RL;
      const bool live = row < rows;
      const int at = row0 + row, qi = at / p.G;
      const int64_t base = (int64_t)(q0 + qi) * p.ldq + ((int64_t)h * p.G + (at - qi * p.G)) * D + c8 * 8;
      float x[8];
      if (live && p.q_vec) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + base));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 f = dt_unpack2(p.qdt, w[k]);
          x[2 * k] = f.x;
          x[2 * k + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = live ? dt_load(p.q, base + k, p.qdt) : 0.f;
      }
      float up = sign, e = 1.f;
      if (p.qdt != WG_DT_F16) {
        float mx = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
        for (int o = 1; o < RL; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (mx > 0.f && mx <= 3.402823466e38f) {
          query_range(mx, &up, &e);
          up *= sign;
        }
      }
      *reinterpret_cast<uint4*>(qs + f_off<D>(row, c8)) =
          make_uint4(pack_f16(x[0] * up, x[1] * up), pack_f16(x[2] * up, x[3] * up), pack_f16(x[4] * up, x[5] * up),
                     pack_f16(x[6] * up, x[7] * up));
      if (c8 == 0) row_mul[row] = e * fabsf(p.scale) * KV8_LOG2E;  // scores in units of log 2
    }
    __syncthreads();
    const uint32_t qu = (uint32_t)__cvta_generic_to_shared(qs);
#pragma unroll
    for (int j = 0; j < KS; j++) ldm4(qf[j], qu + f_off<D>(warp * 16 + (lane & 15), 2 * j + (lane >> 4)));
    mul[0] = row_mul[ra];
    mul[1] = row_mul[rb];
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
  const uint32_t smem_u = (uint32_t)__cvta_generic_to_shared(smem);

  for (int buf = 0; c < c_end; c++, buf ^= 1) {
    uint8_t* kt = smem + buf * 2 * tile_bytes<D>();
    convert(kt, kraw);
    convert(kt + tile_bytes<D>(), vraw);
    if (tid < 4) meta(buf)[tid] = make_float4(sk, sv, ok ? 1.f : 0.f, 0.f);
    __syncthreads();  // the chunk is in place, and everyone is done with the one before the last
    if (c + 1 < c_end) fetch(c + 1);
    if (__all_sync(0xffffffffu, c * PT >= lim_a && c * PT >= lim_b)) continue;  // nothing visible to the warp
    const uint32_t ku = smem_u + buf * 2 * tile_bytes<D>(), vu = ku + tile_bytes<D>();
    const float4* mt = meta(buf);

    // ---- scores
    float s[8][4];
#pragma unroll
    for (int n = 0; n < 8; n++) {
#pragma unroll
      for (int kk = 0; kk < KS / 2; kk++) {
        uint32_t b[4];
        ldm4(b, ku + f_off<D>(n * 8 + (lane & 7), kk * 4 + (lane >> 3)));
        if (kk == 0) mma16816_zero(s[n], qf[0], b[0], b[1]);
        else mma16816(s[n], qf[2 * kk], b[0], b[1]);
        mma16816(s[n], qf[2 * kk + 1], b[2], b[3]);
      }
    }
    bool all_ok = true;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const float4 f = mt[q];
      all_ok &= f.z != 0.f;
#pragma unroll
      for (int n = 2 * q; n < 2 * q + 2; n++) {
        s[n][0] *= f.x * mul[0];
        s[n][1] *= f.x * mul[0];
        s[n][2] *= f.x * mul[1];
        s[n][3] *= f.x * mul[1];
      }
    }
    if ((c + 1) * PT > warp_lo || !all_ok) {
#pragma unroll
      for (int n = 0; n < 8; n++) {
        const int j = c * PT + n * 8 + 2 * t;
        const bool there = mt[n >> 1].z != 0.f;
        if (!there || j >= lim_a) s[n][0] = -INFINITY;
        if (!there || j + 1 >= lim_a) s[n][1] = -INFINITY;
        if (!there || j >= lim_b) s[n][2] = -INFINITY;
        if (!there || j + 1 >= lim_b) s[n][3] = -INFINITY;
      }
    }
    // ---- running maximum
    float x_a = m_a, x_b = m_b;
#pragma unroll
    for (int n = 0; n < 8; n++) {
      x_a = fmaxf(x_a, fmaxf(s[n][0], s[n][1]));
      x_b = fmaxf(x_b, fmaxf(s[n][2], s[n][3]));
    }
    x_a = quad_max(x_a);
    x_b = quad_max(x_b);
    const float ref_a = x_a == -INFINITY ? 0.f : x_a, ref_b = x_b == -INFINITY ? 0.f : x_b;
    if (__any_sync(0xffffffffu, x_a != m_a || x_b != m_b)) {
      const float al_a = ex2(m_a - ref_a), al_b = ex2(m_b - ref_b);
      l_a *= al_a;
      l_b *= al_b;
#pragma unroll
      for (int j = 0; j < NT; j++) {
        o[j][0] *= al_a;
        o[j][1] *= al_a;
        o[j][2] *= al_b;
        o[j][3] *= al_b;
      }
      m_a = x_a;
      m_b = x_b;
    }
    // lifted weights rounded to f16; their sum, by the same MMA over a matrix of
    // ones, is that of the rounded ones
    const float lift_a = KV8_LIFT - ref_a, lift_b = KV8_LIFT - ref_b;
    uint32_t pf[4][4];
#pragma unroll
    for (int n = 0; n < 8; n++) {
      pf[n >> 1][(n & 1) * 2] = pack_weights(ex2(s[n][0] + lift_a), ex2(s[n][1] + lift_a));
      pf[n >> 1][(n & 1) * 2 + 1] = pack_weights(ex2(s[n][2] + lift_b), ex2(s[n][3] + lift_b));
    }
    float rs[4];
    mma16816_zero(rs, pf[0], 0x3c003c00u, 0x3c003c00u);
#pragma unroll
    for (int q = 1; q < 4; q++) mma16816(rs, pf[q], 0x3c003c00u, 0x3c003c00u);
    l_a = fmaf(rs[0], KV8_UNLIFT, l_a);
    l_b = fmaf(rs[2], KV8_UNLIFT, l_b);
    // ---- P.V: the tokens of a page into fresh accumulators, which its scale joins to the sum
#pragma unroll
    for (int q = 0; q < PT / GT; q++) {
      const float f = mt[q * (GT / 16)].y * KV8_UNLIFT;
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        float a0[4], a1[4];
#pragma unroll
        for (int k = 0; k < GT / 16; k++) {
          const int step = q * (GT / 16) + k;
          uint32_t b[4];
          ldm4t(b, vu + f_off<D>(step * 16 + (lane & 15), j + (lane >> 4)));
          if (k == 0) {
            mma16816_zero(a0, pf[step], b[0], b[1]);
            mma16816_zero(a1, pf[step], b[2], b[3]);
          } else {
            mma16816(a0, pf[step], b[0], b[1]);
            mma16816(a1, pf[step], b[2], b[3]);
          }
        }
#pragma unroll
        for (int x = 0; x < 4; x++) {
          o[j][x] = fmaf(f, a0[x], o[j][x]);
          o[j + 1][x] = fmaf(f, a1[x], o[j + 1][x]);
        }
      }
    }
  }

  auto row_at = [&](int row) -> int64_t {  // a row's place in out
    const int at = row0 + row, qi = at / p.G;
    return (int64_t)(q0 + qi) * p.ldo + ((int64_t)h * p.G + (at - qi * p.G)) * D;
  };
  auto store = [&](int64_t at, float x, float y) {
    if (p.o_vec) {
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + at) = dt_pack2(p.odt, x, y);
    } else {
      dt_store(p.out, at, p.odt, x);
      dt_store(p.out, at + 1, p.odt, y);
    }
  };
  auto over = [](float l) { return l > 0.f || l != l ? 1.f / l : 0.f; };  // nothing visible: zeros; NaN stays
  if (p.splits == 1) {
    const float ia = over(l_a), ib = over(l_b);
    const int64_t at_a = row_at(ra) + 2 * t, at_b = row_at(rb) + 2 * t;
    if (ra < rows) {
#pragma unroll
      for (int j = 0; j < NT; j++) store(at_a + j * 8, o[j][0] * ia, o[j][1] * ia);
    }
    if (rb < rows) {
#pragma unroll
      for (int j = 0; j < NT; j++) store(at_b + j * 8, o[j][2] * ib, o[j][3] * ib);
    }
    return;
  }
  // ---- join the cluster's CTAs: O, then m and l, in the tiles' memory
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
  float* ml = sums + PR * D;
#pragma unroll
  for (int j = 0; j < NT; j++) {
    *reinterpret_cast<float2*>(sums + ra * D + j * 8 + 2 * t) = make_float2(o[j][0], o[j][1]);
    *reinterpret_cast<float2*>(sums + rb * D + j * 8 + 2 * t) = make_float2(o[j][2], o[j][3]);
  }
  if (t == 0) {
    ml[ra] = m_a;
    ml[rb] = m_b;
    ml[PR + ra] = l_a;
    ml[PR + rb] = l_b;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  for (int i = tid * p.splits + rank; i < rows * (D / 2); i += PW * 32 * p.splits) {
    const int row = i / (D / 2), d = (i % (D / 2)) * 2;
    float m = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
    for (int k = 0; k < p.splits; k++) {
      const float* po = cl.map_shared_rank(sums, k);
      const float pm = po[PR * D + row], pl = po[PR * D + PR + row];
      const float2 v = *reinterpret_cast<const float2*>(po + row * D + d);
      const float nm = fmaxf(m, pm), ref = nm == -INFINITY ? 0.f : nm;
      const float fo = ex2(m - ref), fn = ex2(pm - ref);
      l = l * fo + pl * fn;
      x = x * fo + v.x * fn;
      y = y * fo + v.y * fn;
      m = nm;
    }
    const float inv = over(l);
    store(row_at(row) + d, x * inv, y * inv);
  }
  cl.sync();  // peers may still be reading this CTA
}

typedef void (*PromptKernel)(const Kv8AttnArgs);
PromptKernel pick(int head_dim, int page) {
  if (head_dim == 64) return page == 16 ? prompt_attn_kernel<64, 16> : page == 32 ? prompt_attn_kernel<64, 32> : prompt_attn_kernel<64, 64>;
  return page == 16 ? prompt_attn_kernel<128, 16> : page == 32 ? prompt_attn_kernel<128, 32> : prompt_attn_kernel<128, 64>;
}

}  // namespace

int kv8_prompt_attributes() {
  for (int d = 64; d <= 128; d += 64)
    for (int page = 16; page <= 64; page *= 2) {
      WG_CHECK_CUDA(cudaFuncSetAttribute(pick(d, page), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         d == 64 ? prompt_smem<64>() : prompt_smem<128>()));
      WG_CHECK_CUDA(cudaFuncSetAttribute(pick(d, page), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    }
  return WG_OK;
}

int launch_kv8_prompt(Kv8AttnArgs a, int head_dim, int64_t max_kv, cudaStream_t st) {
  const int64_t rows = (int64_t)a.max_q * a.G, tiles = (rows + PR - 1) / PR, units = tiles * a.H * a.R;
  const int64_t chunks = (max_kv + PT - 1) / PT;
  // CTAs per tile: enough for two on every SM, none with less than 8 chunks
  int64_t s = (148 * 2 + units - 1) / units;
  if (s > chunks / 8) s = chunks / 8;
  a.splits = (int)(s < 1 ? 1 : s > KV8_MAX_SPLIT ? KV8_MAX_SPLIT : s);
  a.tiles = (int)tiles;
  if (units * a.splits > 0x7fffffffLL) {
    set_error("wg_kv8_attention: %lld CTAs are more than a grid holds", (long long)(units * a.splits));
    return WG_ERR_INVALID;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * a.splits));
  cfg.blockDim = dim3(PW * 32);
  cfg.dynamicSmemBytes = head_dim == 64 ? prompt_smem<64>() : prompt_smem<128>();
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
  return launch_check(cudaLaunchKernelEx(&cfg, pick(head_dim, 1 << a.shift), a), "kv8_prompt");
}

}  // namespace wg
