// Gated delta rule over whole sequences (sm_100a): prompts of any length and
// single tokens, without a tape.  For every sequence n, value head hv (k/q
// head hk = hv / (Hv / Hk)) and step t of the sequence
//     S' = S g_t;  delta = (v_t - S' k_t) beta_t;  S = S' + delta (x) k_t;  y_t = S q_t
// from state_in[n] to state_out[n].  A step whose mask is 0 leaves S as it is
// and writes y = 0; nothing it holds is read into a sum.
//
// Sequences are the rows of a [B, T] batch, or pieces cu[n] .. cu[n+1] of one
// row of T tokens (packed).  Tokens are addressed as base + token * ld + head *
// D, so q, k and v may be slices of one wider projection output.
//
// The reference runs this step for caches that record no tape through
// mlx-lm's gated_delta_update (third party), from the hook at
// dflash_mlx/engine/target_qwen_gdn.py:551-651.

namespace dfl {
namespace gdnr {

struct RuleParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const float* g;
  const float* beta;
  const uint8_t* mask;  // [tokens] or null
  const int32_t* cu;    // [B + 1] or null
  const float* state_in;
  float* state_out;
  __nv_bfloat16* y;
  int ldq, ldk, ldv;  // elements from one token to the next
  int B, T, Hv, Hk, Dv;
  int g_vec;
  int zero_gaps;  // write 0 to the y rows of no sequence (packed)
};

// First token and length of sequence n.  Offsets that decrease or leave
// [0, T] are recorded in the device error word; what they name is cut to the
// range, so every access stays inside the buffers.
__device__ __forceinline__ void sequence_range(const RuleParams& p, int n, size_t* first, int* len) {
  if (!p.cu) {
    *first = (size_t)n * p.T;
    *len = p.T;
    return;
  }
  const int a = p.cu[n], b = p.cu[n + 1];
  const int a1 = min(max(a, 0), p.T);
  const int b1 = min(max(b, a1), p.T);
  if ((a1 != a || b1 != b) && threadIdx.x == 0) atomicExch(&g_device_error, kDevBadInput);
  *first = (size_t)a1;
  *len = b1 - a1;
}

// y rows before the first and behind the last sequence, columns [c0, c0 + cols)
// of value head hv, by the CTAs of those two sequences.
__device__ __forceinline__ void zero_gap_rows(const RuleParams& p, int n, int hv, int c0, int cols) {
  if (!p.cu || !p.zero_gaps || (n != 0 && n != p.B - 1)) return;
  const int first = min(max(p.cu[0], 0), p.T), last = min(max(p.cu[p.B], 0), p.T);
  const int lo = n == 0 ? first : 0;                 // rows [0, lo) ...
  const int hi = n == p.B - 1 ? p.T - last : 0;      // ... and the last hi rows
  const int total = lo + hi;
  for (size_t i = threadIdx.x; i < (size_t)total * cols; i += blockDim.x) {
    const int r = int(i / cols), c = int(i % cols);
    const size_t token = r < lo ? r : size_t(last) + (r - lo);
    p.y[(token * p.Hv + hv) * p.Dv + c0 + c] = __float2bfloat16_rn(0.f);
  }
}

// ------------------------------------------------------------- recurrent form
// One step after the other.  A row of the state is spread over LPR = Dk / 16
// lanes, lane l holding columns 4 (l + LPR i) .. + 3 (i < 4): a row's loads
// and stores are 16 bytes a lane, next to each other, and its two dot products
// end in log2(LPR) shuffles.  A thread owns two rows, which share the k and q
// chunks read from shared memory.  The inputs of up to 16 steps are staged at
// a time; at one token per sequence the kernel is a pass over the state: read
// once, written once.
constexpr int R_THREADS = 128;

template <int DK>
struct RCfg {
  static constexpr int STEPS = DK == 256 ? 8 : 16;           // steps staged at a time (48 KB of shared memory)
  static constexpr int LPR = DK / 16;                        // lanes of a row
  static constexpr int ROWS = 2 * (R_THREADS / LPR);         // rows of a CTA
};

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <int DK, bool GVEC>
__global__ void __launch_bounds__(R_THREADS) gdn_rule_recurrent(const RuleParams p) {
  using C = RCfg<DK>;
  constexpr int LPR = C::LPR;
  constexpr int R_STEPS = C::STEPS;
  __shared__ __align__(16) float k_s[R_STEPS][DK];
  __shared__ __align__(16) float q_s[R_STEPS][DK];
  __shared__ __align__(16) float gv_s[GVEC ? R_STEPS : 1][GVEC ? DK : 4];
  __shared__ float v_s[R_STEPS][C::ROWS];
  __shared__ float g_s[R_STEPS], b_s[R_STEPS];
  __shared__ int m_s[R_STEPS];

  const int blocks_per_head = (p.Dv + C::ROWS - 1) / C::ROWS;
  const int nh = blockIdx.x / blocks_per_head;  // n * Hv + hv
  const int row0 = (blockIdx.x - nh * blocks_per_head) * C::ROWS;
  const int n = nh / p.Hv;
  const int hv = nh - n * p.Hv;
  const int hk = hv / (p.Hv / p.Hk);
  size_t first;
  int len;
  sequence_range(p, n, &first, &len);
  zero_gap_rows(p, n, hv, row0, min(C::ROWS, p.Dv - row0));

  const int lane = threadIdx.x % LPR;
  const int r0 = 2 * (threadIdx.x / LPR);   // rows r0, r0 + 1 of the CTA
  const bool live = row0 + r0 < p.Dv;       // Dv is even: both rows or none
  const size_t off = (size_t)nh * p.Dv * DK + (size_t)(row0 + r0) * DK + 4 * lane;
  float s[2][16];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = live ? *reinterpret_cast<const float4*>(p.state_in + off + j * DK + 4 * LPR * i)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
      s[j][4 * i] = x.x; s[j][4 * i + 1] = x.y; s[j][4 * i + 2] = x.z; s[j][4 * i + 3] = x.w;
    }

  for (int t0 = 0; t0 < len; t0 += R_STEPS) {
    const int steps = min(R_STEPS, len - t0);
    if (t0) __syncthreads();
    for (int i = threadIdx.x; i < steps * DK; i += R_THREADS) {
      const int t = i / DK, d = i % DK;
      const size_t token = first + t0 + t;
      k_s[t][d] = __bfloat162float(p.k[token * p.ldk + (size_t)hk * DK + d]);
      q_s[t][d] = __bfloat162float(p.q[token * p.ldq + (size_t)hk * DK + d]);
      if constexpr (GVEC) gv_s[t][d] = p.g[(token * p.Hv + hv) * DK + d];
    }
    for (int i = threadIdx.x; i < steps * C::ROWS; i += R_THREADS) {
      const int t = i / C::ROWS, r = i % C::ROWS;
      if (row0 + r < p.Dv)
        v_s[t][r] = __bfloat162float(p.v[(first + t0 + t) * p.ldv + (size_t)hv * p.Dv + row0 + r]);
    }
    if (threadIdx.x < steps) {
      const size_t token = first + t0 + threadIdx.x;
      if constexpr (!GVEC) g_s[threadIdx.x] = p.g[token * p.Hv + hv];
      b_s[threadIdx.x] = p.beta[token * p.Hv + hv];
      m_s[threadIdx.x] = p.mask ? p.mask[token] != 0 : 1;
    }
    __syncthreads();
    for (int t = 0; t < steps; ++t) {
      const size_t out = ((first + t0 + t) * p.Hv + hv) * p.Dv + row0 + r0;
      if (!m_s[t]) {
        if (lane == 0 && live)
          *reinterpret_cast<__nv_bfloat162*>(p.y + out) = __floats2bfloat162_rn(0.f, 0.f);
        continue;
      }
      float kt[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(&k_s[t][4 * (lane + LPR * i)]);
        kt[4 * i] = x.x; kt[4 * i + 1] = x.y; kt[4 * i + 2] = x.z; kt[4 * i + 3] = x.w;
      }
      float a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float gt = GVEC ? gv_s[t][4 * (lane + LPR * (i / 4)) + i % 4] : g_s[t];
        s[0][i] *= gt;
        s[1][i] *= gt;
        a0 = __fmaf_rn(s[0][i], kt[i], a0);
        a1 = __fmaf_rn(s[1][i], kt[i], a1);
      }
      const float d0 = (v_s[t][r0] - row_sum<LPR>(a0)) * b_s[t];
      const float d1 = (v_s[t][r0 + 1] - row_sum<LPR>(a1)) * b_s[t];
      float y0 = 0.f, y1 = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(&q_s[t][4 * (lane + LPR * i)]);
        const float qt[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[0][4 * i + e] = __fmaf_rn(kt[4 * i + e], d0, s[0][4 * i + e]);
          s[1][4 * i + e] = __fmaf_rn(kt[4 * i + e], d1, s[1][4 * i + e]);
          y0 = __fmaf_rn(s[0][4 * i + e], qt[e], y0);
          y1 = __fmaf_rn(s[1][4 * i + e], qt[e], y1);
        }
      }
      y0 = row_sum<LPR>(y0);
      y1 = row_sum<LPR>(y1);
      if (lane == 0 && live)
        *reinterpret_cast<__nv_bfloat162*>(p.y + out) = __floats2bfloat162_rn(y0, y1);
    }
  }

  if (live) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(p.state_out + off + j * DK + 4 * LPR * i) =
            make_float4(s[j][4 * i], s[j][4 * i + 1], s[j][4 * i + 2], s[j][4 * i + 3]);
  }
}

template <int DK>
int launch_recurrent(const RuleParams& p, cudaStream_t stream) {
  const long long grid = (long long)p.B * p.Hv * ((p.Dv + RCfg<DK>::ROWS - 1) / RCfg<DK>::ROWS);
  if (grid > 0x7fffffffll) return DFL_ERR_BAD_SHAPE;
  int dev, sms;
  const int st = host::current_device(&dev, &sms);
  if (st != DFL_OK) return st;
  if (p.g_vec)
    gdn_rule_recurrent<DK, true><<<int(grid), R_THREADS, 0, stream>>>(p);
  else
    gdn_rule_recurrent<DK, false><<<int(grid), R_THREADS, 0, stream>>>(p);
  return host::launch_status();
}

// Checks shared by the two forms; fills *p.  *done: nothing to launch.
inline int rule_params(const uint16_t* q, int ldq, const uint16_t* k, int ldk, const uint16_t* v, int ldv,
                       const float* g, int g_vec, const float* beta, const uint8_t* mask,
                       const int32_t* cu, const float* state_in, float* state_out, uint16_t* y,
                       int zero_gaps, int B, int T, int Hv, int Hk, int Dv, int Dk, RuleParams* p,
                       bool* done) {
  *done = false;
  if (B < 0 || T < 0 || Hv < 1 || Hk < 1 || Hv % Hk != 0 || Dv < 32 || Dv % 32 != 0)
    return DFL_ERR_BAD_SHAPE;
  if (Dk != 32 && Dk != 64 && Dk != 128 && Dk != 256) return DFL_ERR_BAD_SHAPE;
  if ((long long)Hk * Dk > 0x7fffffffll || (long long)Hv * Dv > 0x7fffffffll) return DFL_ERR_BAD_SHAPE;
  if (ldq < Hk * Dk || ldk < Hk * Dk || ldv < Hv * Dv) return DFL_ERR_BAD_SHAPE;
  if (B == 0) {
    *done = true;
    return DFL_OK;
  }
  if (!state_in || !state_out) return DFL_ERR_NULL_POINTER;
  if (T > 0 && (!q || !k || !v || !g || !beta || !y)) return DFL_ERR_NULL_POINTER;
  if (!host::aligned(state_in, 16) || !host::aligned(state_out, 16) || !host::aligned(y, 16))
    return DFL_ERR_MISALIGNED;
  p->q = reinterpret_cast<const __nv_bfloat16*>(q);
  p->k = reinterpret_cast<const __nv_bfloat16*>(k);
  p->v = reinterpret_cast<const __nv_bfloat16*>(v);
  p->g = g;
  p->beta = beta;
  p->mask = mask;
  p->cu = cu;
  p->state_in = state_in;
  p->state_out = state_out;
  p->y = reinterpret_cast<__nv_bfloat16*>(y);
  p->ldq = ldq;
  p->ldk = ldk;
  p->ldv = ldv;
  p->B = B;
  p->T = T;
  p->Hv = Hv;
  p->Hk = Hk;
  p->Dv = Dv;
  p->g_vec = g_vec ? 1 : 0;
  p->zero_gaps = zero_gaps ? 1 : 0;
  return DFL_OK;
}

}  // namespace gdnr
}  // namespace dfl

extern "C" int dfl_gdn_rule_recurrent(const uint16_t* q, int ldq, const uint16_t* k, int ldk,
                                      const uint16_t* v, int ldv, const float* g, int g_vectorized,
                                      const float* beta, const uint8_t* mask, const int32_t* cu_seqlens,
                                      const float* state_in, float* state_out, uint16_t* y, int zero_gaps,
                                      int B, int T, int Hv, int Hk, int Dv, int Dk, void* stream) {
  using namespace dfl;
  gdnr::RuleParams p;
  bool done;
  const int st = gdnr::rule_params(q, ldq, k, ldk, v, ldv, g, g_vectorized, beta, mask, cu_seqlens, state_in,
                                   state_out, y, zero_gaps, B, T, Hv, Hk, Dv, Dk, &p, &done);
  if (st != DFL_OK || done) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (Dk) {
    case 32: return gdnr::launch_recurrent<32>(p, s);
    case 64: return gdnr::launch_recurrent<64>(p, s);
    case 128: return gdnr::launch_recurrent<128>(p, s);
    default: return gdnr::launch_recurrent<256>(p, s);
  }
}
