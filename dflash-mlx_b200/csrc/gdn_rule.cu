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
// once, written once.  40 tokens of 48 heads of 128 x 128 (253 MB) take 54 us,
// 71% of the measured copy rate; one token 3.9 us, launch and one trip to
// memory.  Over more steps it is bound by fp32 arithmetic and the shuffles: 0.5
// us a step of one sequence of 48 heads.
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

// --------------------------------------------------------------- chunked form
// Steps are taken 64 at a time.  With D_ij = g_{j+1} .. g_i (1 for i = j),
// c_i = g_0 .. g_i, S the state before the chunk and K, Q, V the chunk's rows,
//     A_ij = beta_i D_ij (k_i . k_j) for j < i, else 0,   T = (I + A)^-1,
//     R = diag(beta) (V - diag(c) K S^T),                 Delta = T R,
//     Y = diag(c) Q S^T + P Delta,  P_ij = D_ij (q_i . k_j) for j <= i,
//     S <- c_63 S + sum_i D_63,i delta_i (x) k_i
// is what the 64 steps give one after the other.  D is formed by products, not
// as a quotient or an exponential of sums, so decays of 0 or of any size are
// exact cases.
//
// A CTA owns up to 128 value rows of one head and walks the sequence's chunks.
// All products run on the tensor cores transposed, value rows in the 128 TMEM
// lanes: S K^T, S Q^T, R T^T, Delta P^T and Delta K, so the state row, R and
// Delta of a value row stay with its threads (fp32 in registers), enter the
// products from TMEM, and only K, Q, T and P are read from shared memory, K
// both as it is and transposed from the same tile.
//
// fp32 in bf16 products: K and Q are bf16 already.  The state, R, T - I and the
// update Delta K go in as three bf16 parts (24 bits), and T is joined from 32-bit
// blocks, so what is carried from chunk to chunk keeps 32-bit accuracy (T - I in
// two parts would do only for keys at right angles: it is as large as R's own
// share where they are alike).  The tensor cores cut their sums to 24 bits, so
// the small parts' products are added up before the large ones.  State error
// (2-norm) of 520 steps of slow decay, keys of unit length, against 64 bits: 1.3e-7
// at a mean cosine of 0 between keys, 1.8e-7 at 0.5, 2.7e-7 at 0.95, 4.4e-7 there
// with beta near 1; cut in pieces 3e-7 to 8e-7; a recurrence in fp32 2e-7.  In y,
// which ends in 8 bits, the state, P and Delta have two parts (one each of P and
// Delta would add 2.2e-3 of y to the 1.7e-3 of its last rounding).
//
// Bound by the work on a chunk, not by a rate.  The preparing warps take 11000
// cycles for T and P of the next chunk (decays 3700, blocks of 16 inverted 1700,
// joined 5300, a third of it for 32-bit factors), and beside them the chain through a
// chunk takes 9700: S K^T, R, R T^T, Delta, Delta K and the new state wait for one
// another.  Most of that is the state's threads at work: 3000 cycles on the last
// chunk's y, 700 on R, 1000 on Delta, 2100 on beta V, 1500 on the state; they wait
// 1800 for products, and 1200 to 1600 for T.  A chunk of a 128 x 128 head takes 6.1 us
// (11200 cycles) with an SM of each pair idle, 6.4 to 7.1 with every SM at work (two
// share their instruction fetches).  A CTA's start and end take 9 us more.  8192 steps
// of 48 heads, cut in three, 612 us; 15886 steps in 8 prompts 596 us.
//
// Warps: 0-3 prepare T and P of the next chunk (K K^T and Q K^T from one
// product, inverse by blocks of 16, 32 and 64 in fp32) and put zeros over rows
// of masked steps and behind the end; 4-11 (two threads per value row, half the
// columns each) carry the state; 12 and 14 issue the products and 13
// the loads (TMA, two chunks ahead); 15 only lends its registers.
constexpr int CH = 64;               // steps of a chunk
constexpr int C_THREADS = 16 * 32;
// Registers of a thread after the split; the launch has 128 for each, and
// 96 + 2 x 184 + 48 = 4 x 128.
constexpr int C_REGS_PREP = 96, C_REGS_STATE = 184, C_REGS_ISSUE = 48;
constexpr int C_ORDER = 256;         // packed sequences that are taken longest first
constexpr int C_STAGES = 3;
constexpr int C_PREP = 128, C_STATE = 256;
// A in fp32, floats of a row and of a block: blocks 0-3 on the diagonal (16 x
// 16), 4 and 5 left of blocks 1 and 3, then the 32 x 32 block at (32, 0).
constexpr int DIAG_LD = 20, DIAG_BLK = 16 * DIAG_LD + 4, OFF_LD = 36;
constexpr int A32_FLOATS = 6 * DIAG_BLK + 32 * OFF_LD;
constexpr int PART = CH * 128;       // bytes of one bf16 part of a 64 x 64 matrix, 128-byte swizzle

template <int DK>
struct CCfg {
  static constexpr int ATOM = 128 * 128;                 // 128 rows (K, then Q) x 64 columns
  static constexpr int KQ_BYTES = (DK / 64) * ATOM;
  static constexpr int V_BYTES = CH * 256;               // 64 rows x 128 columns
  static constexpr int V_OFF = C_STAGES * KQ_BYTES;      // of two chunks
  static constexpr int TP_BYTES = 5 * PART;              // T's three parts and P's two
  static constexpr int TP_OFF = V_OFF + 2 * V_BYTES;
  static constexpr int A_OFF = TP_OFF + 2 * TP_BYTES;    // A in fp32, a place for stores to nowhere
  static constexpr int SMALL_OFF = A_OFF + A32_FLOATS * 4 + 1024;
  static constexpr int SMALL_BYTES = (C_STAGES * 2 + 2 * 3) * CH * 4;
  static constexpr int SMEM_BYTES = SMALL_OFF + SMALL_BYTES + 1024;
  static_assert(SMEM_BYTES + 1024 <= 227 * 1024, "with the barriers, what a CTA can have");
  // TMEM columns
  static constexpr int S_PART = DK / 2;                  // columns of one part of the state
  static constexpr int COL_S = 0;                        // state parts; later Delta K's three parts
  static constexpr int COL_D = 192;                      // S K^T, then R T^T, then Delta K
  static constexpr int COL_G = 256;                      // [K; Q] K^T, over Delta K's second half
  static constexpr int COL_SQ = 320;                     // S Q^T
  static constexpr int COL_R = 384;                      // R's parts, then Delta
  static constexpr int COL_Y = 448;                      // R's third part, later Delta P^T
  // R's third part of 16 steps: each half over its own warps' half of y, which
  // they have read
  static __host__ __device__ constexpr int col_r3(int k) { return COL_Y + (k / 2) * 32 + (k % 2) * 8; }
};

// mbar_wait_abortable in few instructions (32 bits of the clock): there are
// thirty waits below, and with two SMs at work behind one instruction cache a
// chunk's code has to stay small (unrolled all through, a third of the cycles
// went on fetching it).
__device__ __forceinline__ void wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_word) {
  if (mbar_try_wait(bar, parity)) return;
  uint32_t t0, t1;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t0));
#pragma unroll 1
  while (!*abort_word && !mbar_try_wait(bar, parity)) {
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t1));
    if (t1 - t0 > uint32_t(kWaitLimitNs)) {
      atomicExch(&g_device_error, kDevWaitTimeout);
      *abort_word = 1;
    }
  }
}

// The leading bf16 parts of two values; what they leave stays in a, b (exact).
__device__ __forceinline__ uint32_t take_part(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
  asm("{\n\t.reg .b64 x, y, m;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%0, %1};\n\t"
      "mov.b64 m, 0xbf800000bf800000;\n\t"
      "fma.rn.f32x2 y, x, m, y;\n\t"
      "mov.b64 {%0, %1}, y;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(__uint_as_float(u << 16)), "f"(__uint_as_float(u & 0xffff0000u)));
  return u;
}

// The leading parts of eight values, as the 16 bytes that they take in a part.
__device__ __forceinline__ uint4 take_part8(float* x) {
  uint4 u;
  u.x = take_part(x[0], x[1]);
  u.y = take_part(x[2], x[3]);
  u.z = take_part(x[4], x[5]);
  u.w = take_part(x[6], x[7]);
  return u;
}

// (d0, d1) = (a0, a1) * (b0, b1) + (c0, c1), one packed instruction
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0,
                                     float c1) {
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %5};\n\t"
      "mov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

template <int REGS>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

template <int REGS>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// The parts of 16 values into 8 TMEM columns each, at the given addresses.
template <int PARTS>
__device__ __forceinline__ void store_parts(const uint32_t (&taddr)[PARTS], float (&x)[16]) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = take_part(x[2 * i], x[2 * i + 1]);
    tmem_st_32x32b_x8(taddr[p], u);
  }
}

struct ChunkBars {
  uint64_t loaded[C_STAGES], full[C_STAGES], v_loaded[2];
  uint64_t tp_full[2], tp_freed[2];
  uint64_t g_full, g_read;
  uint64_t s_ready, d1_done, r_ready, d3_done, delta_ready, d4_done, q_done, y_done, y_read;
};

__device__ __forceinline__ float4 at4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 v = at4(p + i);
    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
  }
}

// Byte offset of element (r, c) in a part of a 64 x 64 matrix.
__device__ __forceinline__ int part_at(int r, int c) { return r * 128 + (((c / 8) ^ (r & 7)) * 16) + (c % 8) * 2; }

// Inverse of a unit lower triangular block of 16 rows (strictly lower part
// used) by forward substitution, in place, column c per lane, 16 lanes of one
// warp a block.
__device__ __forceinline__ void invert_block16(float* blk, int c) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float s0 = i == c ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < i; j += 4) {
      const float4 m = at4(blk + i * DIAG_LD + j);
      s0 = __fmaf_rn(-m.x, x[j], s0);
      if (j + 1 < i) s1 = __fmaf_rn(-m.y, x[j + 1], s1);
      if (j + 2 < i) s0 = __fmaf_rn(-m.z, x[j + 2], s0);
      if (j + 3 < i) s1 = __fmaf_rn(-m.w, x[j + 3], s1);
    }
    x[i] = s0 + s1;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) blk[i * DIAG_LD + c] = x[i];
}

// Row 16 b + c of T - I in its diagonal block, in parts.
__device__ __forceinline__ void store_diag_row(const float* diag, uint8_t* t, int b, int c) {
  float x[16];
  load16(diag + b * DIAG_BLK + c * DIAG_LD, x);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = i == c ? 0.f : x[i];
  uint8_t* at0 = t + part_at(16 * b + c, 16 * b);
  uint8_t* at1 = t + part_at(16 * b + c, 16 * b + 8);
#pragma unroll 1
  for (int part = 0; part < 3; ++part) {
    *reinterpret_cast<uint4*>(at0 + part * PART) = take_part8(x);
    *reinterpret_cast<uint4*>(at1 + part * PART) = take_part8(x + 8);
  }
}

// x as two numbers of 11 bits, what a factor of a tf32 product can hold: rounded,
// and what that leaves, cut (together they are off by 2^-23 of x at most).  A NaN
// stays one in the second.
__device__ __forceinline__ void two_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

__device__ __forceinline__ void mma_m16n8k8(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// acc + low (16 rows, NT tiles of 8 columns) += A B over 8 k's.  x: A's rows lane / 4
// and + 8, k's 2 (lane % 4) and + 1 (row by row); b: this lane's column lane / 4 of row 2
// (lane % 4) of B's first tile.  The instruction's k's 0-3 and 4-7 stand for the even
// and the odd ones, so that A's come as pairs, an accumulator's as they lie.  First x
// first goes to acc, first x second and second x first, which are small, to low; the
// part left out is 2^-22 of a factor.  Each over the tiles in turn, so that neighbours
// do not wait for one another.
template <int NT, int LD>
__device__ __forceinline__ void mma_tf32(float (*acc)[4], float (*low)[4], const float (&x)[4], const float* b) {
  uint32_t a[2][4], f[2][NT][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) two_tf32(x[i], a[0][(i & 1) * 2 + i / 2], a[1][(i & 1) * 2 + i / 2]);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) two_tf32(b[e * LD + 8 * i], f[0][i][e], f[1][i][e]);
#pragma unroll
  for (int m = 0; m < 3; ++m)
#pragma unroll
    for (int i = 0; i < NT; ++i) mma_m16n8k8(m == 1 ? acc[i] : low[i], a[m == 2], f[m == 0][i]);
}

template <int NT>
__device__ __forceinline__ void add_low(float (&acc)[NT][4], const float (&low)[NT][4]) {
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] += low[i][e];
}

__device__ __forceinline__ void load_rows(const float* a, float (&x)[4]) {   // rows of DIAG_LD
  const float2 u = *reinterpret_cast<const float2*>(a), v = *reinterpret_cast<const float2*>(a + 8 * DIAG_LD);
  x[0] = u.x; x[1] = u.y; x[2] = v.x; x[3] = v.y;
}

// Rows r .. r + 15, columns c .. c + 15 of T, from accumulators, in parts.
__device__ __forceinline__ void store_join(uint8_t* t, float (&out)[2][4], int r, int c, int lane) {
#pragma unroll 1
  for (int part = 0; part < 3; ++part, t += PART)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; e += 2)
        *reinterpret_cast<uint32_t*>(t + part_at(r + lane / 4 + 4 * e, c + 8 * i + 2 * (lane % 4))) =
            take_part(out[i][e], out[i][e + 1]);
}

// T21 = -(T22 A21) T11 for blocks of 16 rows, pair w (rows 32 w + 16 ..): A21 in
// block 4 + w, which T21 goes over, T22 and T11 in blocks 2 w + 1 and 2 w.  The first
// product's accumulators are the second one's left operand in place.
__device__ __forceinline__ void join16(float* diag, uint8_t* t, int w, int lane) {
  const int at_a = (lane / 4) * DIAG_LD + 2 * (lane % 4), at_b = 2 * (lane % 4) * DIAG_LD + lane / 4;
  float* off = diag + (4 + w) * DIAG_BLK;
  const float* t22 = diag + (2 * w + 1) * DIAG_BLK + at_a;
  const float* t11 = diag + 2 * w * DIAG_BLK + at_b;
  float m[2][4] = {}, out[2][4] = {}, ml[2][4] = {}, ol[2][4] = {};
#pragma unroll 1
  for (int k = 0; k < 16; k += 8) {
    float x[4];
    load_rows(t22 + k, x);
    mma_tf32<2, DIAG_LD>(m, ml, x, off + at_b + k * DIAG_LD);
  }
  add_low(m, ml);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float x[4] = {-m[k][0], -m[k][1], -m[k][2], -m[k][3]};
    mma_tf32<2, DIAG_LD>(out, ol, x, t11 + 8 * k * DIAG_LD);
  }
  add_low(out, ol);
  __syncwarp();   // A21 has been read
  float* to = off + at_a;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; e += 2)
      *reinterpret_cast<float2*>(to + 4 * e * DIAG_LD + 8 * i) = make_float2(out[i][e], out[i][e + 1]);
  store_join(t, out, 32 * w + 16, 32 * w, lane);
}

// The same for blocks of 32: rows 32 + r0 .., columns c0 .. of T by a warp, A21 in
// off32, T22 and T11 each in two diagonal blocks and the one left of the lower.  What
// is 0 above the diagonals is passed over: the second 16 k's of the first product
// for r0 = 0, the first 16 of the second for c0 = 16.
__device__ __forceinline__ void join32(const float* diag, const float* off32, uint8_t* t, int r0, int c0, int lane) {
  const int at_a = (lane / 4) * DIAG_LD + 2 * (lane % 4), at_b = 2 * (lane % 4) * DIAG_LD + lane / 4;
  const float* a21 = off32 + 2 * (lane % 4) * OFF_LD + lane / 4;
  float m[4][4] = {}, out[2][4] = {}, ml[4][4] = {}, ol[2][4] = {};
#pragma unroll 1
  for (int k = 0; k < 16 + r0; k += 8) {
    // rows 32 + r0 ..: block 2 for r0 = 0, else block 5 and then 3
    const float* t22 = diag + (r0 == 0 ? 2 : (k < 16 ? 5 : 3)) * DIAG_BLK + at_a + (k & 8);
    float x[4];
    load_rows(t22, x);
    mma_tf32<4, OFF_LD>(m, ml, x, a21 + k * OFF_LD);
  }
  add_low(m, ml);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (8 * k < c0) continue;
    // columns c0 ..: blocks 0 and 4 for c0 = 0, else block 1
    const float* t11 = diag + (c0 != 0 ? 1 : (k < 2 ? 0 : 4)) * DIAG_BLK + at_b + (k & 1) * 8 * DIAG_LD;
    const float x[4] = {-m[k][0], -m[k][1], -m[k][2], -m[k][3]};
    mma_tf32<2, DIAG_LD>(out, ol, x, t11);
  }
  add_low(out, ol);
  store_join(t, out, 32 + r0, c0, lane);
}

// A long sequence cut in n pieces, where there are too few heads to fill the
// card.  A state row s goes through a piece as s -> s M + (what the piece's
// values add), M [Dk, Dk] the same for every row.  First launch: piece 0 whole;
// of pieces 1 .. n - 2 what they make of a zero state (N) and, with the values
// left out, of the unit rows (M).  Then the pieces' first states in turn, S_{i+1} =
// S_i M_i + N_i (chain kernel), and a launch of pieces 1 .. n - 1 from those.  Two
// pieces' time in place of n, for 2 n - 3 CTAs a head.
struct Split {
  int n;         // pieces (1: not cut)
  int last;      // 0: first launch, 1: the one after the chain
  int jobs;      // CTAs of a head
  float* start;  // [heads][n - 1][Dv][Dk] first states of pieces 1 ..
  float* add;    // [heads][n - 2][Dv][Dk] N of pieces 1 .. n - 2
  float* map;    // [heads][n - 2][Dk][Dk] M
};
constexpr int MAX_PIECES = 16;
constexpr int CHAIN_ROWS = 16;

// start[i + 1] = start[i] map[i] + add[i] over the pieces: 16 rows of a head per
// CTA, kept in shared memory; a thread has a column of 8 of them.  The next map
// is copied to shared memory while one is worked with (read from L2 as it is
// needed, a step took 10 us for 2).
template <int DK>
__global__ void __launch_bounds__(2 * DK) gdn_rule_chain(const Split sp, int Dv) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int R = CHAIN_ROWS / 2;
  float* maps = reinterpret_cast<float*>(smem_raw);                                  // [2][DK][DK]
  float(*s)[DK] = reinterpret_cast<float(*)[DK]>(maps + 2 * DK * DK);                // [CHAIN_ROWS][DK]
  const int blocks = Dv / CHAIN_ROWS;
  const size_t head = blockIdx.x / blocks;
  const int row0 = (blockIdx.x % blocks) * CHAIN_ROWS;
  const int c = threadIdx.x % DK, r0 = (threadIdx.x / DK) * R;
  float* start = sp.start + head * (sp.n - 1) * Dv * DK + (size_t)row0 * DK;
  auto fetch = [&](int k) {
    const float* m = sp.map + (head * (sp.n - 2) + k) * DK * DK;
    const uint32_t to = smem_u32(maps + (k & 1) * DK * DK);
    for (int i = threadIdx.x; i < DK * DK / 4; i += 2 * DK) cp_async_16(to + i * 16, m + 4 * i, 16);
    cp_async_commit();
  };
  fetch(0);
#pragma unroll
  for (int i = 0; i < R; ++i) s[r0 + i][c] = start[(size_t)(r0 + i) * DK + c];
  for (int k = 0; k < sp.n - 2; ++k) {
    const float* m = maps + (k & 1) * DK * DK + c;
    const float* add = sp.add + (head * (sp.n - 2) + k) * Dv * DK + (size_t)row0 * DK;
    float acc[R];
#pragma unroll
    for (int i = 0; i < R; ++i) acc[i] = add[(size_t)(r0 + i) * DK + c];
    cp_async_wait_all();
    __syncthreads();   // the map, and the rows
    if (k + 1 < sp.n - 2) fetch(k + 1);
#pragma unroll 4
    for (int j = 0; j < DK; j += 4) {
      const float m0 = m[j * DK], m1 = m[(j + 1) * DK], m2 = m[(j + 2) * DK], m3 = m[(j + 3) * DK];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(&s[r0 + i][j]);
        acc[i] = __fmaf_rn(y.x, m0, acc[i]);
        acc[i] = __fmaf_rn(y.y, m1, acc[i]);
        acc[i] = __fmaf_rn(y.z, m2, acc[i]);
        acc[i] = __fmaf_rn(y.w, m3, acc[i]);
      }
    }
    __syncthreads();
    float* next = start + (size_t)(k + 1) * Dv * DK;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[r0 + i][c] = acc[i];
      next[(size_t)(r0 + i) * DK + c] = acc[i];
    }
  }
}

template <int DK>
constexpr int chain_smem() { return (2 * DK * DK + CHAIN_ROWS * DK) * int(sizeof(float)); }

template <int DK>
__global__ void __launch_bounds__(C_THREADS, 1)
    gdn_rule_chunked(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const RuleParams p, const Split sp) {
  using C = CCfg<DK>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ ChunkBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  __shared__ int chosen;

  const int tiles = (p.Dv + 127) / 128;
  const int job = blockIdx.x % sp.jobs;
  const int hv = (blockIdx.x / sp.jobs) % p.Hv;
  int n = blockIdx.x / (sp.jobs * p.Hv);
  // the piece of the sequence, the value rows, and whether unit rows take their place
  const bool unit = !sp.last && job >= tiles * max(sp.n - 1, 1);
  const int piece = unit ? 1 + job - tiles * (sp.n - 1) : sp.last + job / tiles;
  const int dv0 = unit ? 0 : (job % tiles) * 128;
  const bool partial = unit || (!sp.last && piece > 0);   // N or M: no y
  if (p.cu && p.B > 1 && p.B <= C_ORDER) {
    // Longest sequences first: a CTA's time goes by its chunks, and a long one
    // that starts late would run on alone.
    const int t = threadIdx.x;
    int* lens = reinterpret_cast<int*>(smem_raw);
    if (t < p.B) lens[t] = p.cu[t + 1] - p.cu[t];
    __syncthreads();
    if (t < p.B) {
      int rank = 0;
      for (int u = 0; u < p.B; ++u) rank += lens[u] > lens[t] || (lens[u] == lens[t] && u < t);
      if (rank == n) chosen = t;
    }
    __syncthreads();
    n = chosen;
  }
  const int nh = n * p.Hv + hv;
  const int hk = hv / (p.Hv / p.Hk);
  const int cols = unit ? DK : min(128, p.Dv - dv0);  // value rows of this CTA
  size_t first;
  int len;
  sequence_range(p, n, &first, &len);
  if (piece == 0) zero_gap_rows(p, n, hv, dv0, cols);
  const size_t head = (size_t)p.Dv * DK, row_off = (size_t)dv0 * DK;
  const float* src = p.state_in + nh * head + row_off;   // null: zero (or unit) rows
  float* dst = p.state_out + nh * head + row_off;        // null: not kept
  if (sp.n > 1) {
    const int size = ((len + CH - 1) / CH + sp.n - 1) / sp.n * CH;   // whole chunks
    const int from = min(len, piece * size);
    len = min(len, from + size) - from;
    first += from;
    if (partial) {
      src = nullptr;
      const size_t at = (size_t)nh * (sp.n - 2) + piece - 1;
      dst = unit ? sp.map + at * DK * DK : sp.add + at * head + row_off;
    } else {
      if (piece > 0) src = sp.start + ((size_t)nh * (sp.n - 1) + piece - 1) * head + row_off;
      if (piece < sp.n - 1) dst = piece == 0 ? sp.start + (size_t)nh * (sp.n - 1) * head + row_off : nullptr;
    }
  }
  const int chunks = (len + CH - 1) / CH;
  if (chunks == 0) {
    if (dst && dst != src)
      for (int i = threadIdx.x; i < cols * DK / 4; i += C_THREADS) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (src) {
          x = at4(src + 4 * i);
        } else if (unit) {
          const int r = 4 * i / DK, c = 4 * i % DK;
          x = make_float4(r == c, r == c + 1, r == c + 2, r == c + 3);
        }
        *reinterpret_cast<float4*>(dst + 4 * i) = x;
      }
    return;
  }

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem);
  float* small = reinterpret_cast<float*>(smem + C::SMALL_OFF);
  // g and beta of a stage; c_i, D_63,i and -beta_i c_i of a prepared chunk
  auto g_of = [&](int s) { return small + s * 2 * CH; };
  auto b_of = [&](int s) { return small + s * 2 * CH + CH; };
  auto cum_of = [&](int s) { return small + C_STAGES * 2 * CH + s * 3 * CH; };
  auto until_of = [&](int s) { return small + C_STAGES * 2 * CH + s * 3 * CH + CH; };
  auto nbc_of = [&](int s) { return small + C_STAGES * 2 * CH + s * 3 * CH + 2 * CH; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C_STAGES; ++s) {
      mbar_init(&bars.loaded[s], 1);
      mbar_init(&bars.full[s], C_PREP);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.v_loaded[s], 1);
      mbar_init(&bars.tp_full[s], C_PREP);
      mbar_init(&bars.tp_freed[s], 1 + C_STATE / 32);
    }
    mbar_init(&bars.g_full, 1);
    mbar_init(&bars.g_read, C_PREP);
    mbar_init(&bars.s_ready, C_STATE);
    mbar_init(&bars.d1_done, 1);
    mbar_init(&bars.r_ready, C_STATE);
    mbar_init(&bars.d3_done, 1);
    mbar_init(&bars.delta_ready, C_STATE);
    mbar_init(&bars.d4_done, 1);
    mbar_init(&bars.q_done, 1);
    mbar_init(&bars.y_done, 1);
    mbar_init(&bars.y_read, C_STATE);
    abort_word = 0;
    fence_barrier_init();
  }
  // T and P above their diagonal blocks stay 0; the rest is written per chunk
  for (int i = threadIdx.x; i < 2 * C::TP_BYTES / 16; i += C_THREADS)
    *reinterpret_cast<uint4*>(smem + C::TP_OFF + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_shared();
  if (warp == 12) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint64_t* bar, int parity) {
    wait_on(bar, uint32_t(parity & 1), &abort_word);
  };

  if (warp < 4) {
    // ---------------------------------------------------------- preparation
    fewer_registers<C_REGS_PREP>();
    const int t = threadIdx.x;
    // Chunk c's tiles have landed: zeros over rows of no step, g and beta (1
    // and 0 there: a step that changes nothing) beside them.
    bool on;
    float gv, bv;
    auto fetch = [&](int c) {   // step t / 2 of the chunk
      const size_t tok = first + (size_t)c * CH + t / 2;
      on = t / 2 < len - c * CH && (!p.mask || p.mask[tok] != 0);
      gv = on ? p.g[tok * p.Hv + hv] : 1.f;
      bv = on ? p.beta[tok * p.Hv + hv] : 0.f;
    };
    auto publish = [&](int c) {
      const int s = c % C_STAGES, r = t / 2;
      if (t % 2 == 0) {
        g_of(s)[r] = gv;
        b_of(s)[r] = bv;
      }
      wait(&bars.loaded[s], c / C_STAGES);
      if (!on) {
        uint8_t* kq = smem + s * C::KQ_BYTES;
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (int x = 0; x < DK / 8; ++x)   // one of the row's K and Q per thread
          *reinterpret_cast<uint4*>(kq + (x / 8) * C::ATOM + ((t % 2) * 64 + r) * 128 + (x % 8) * 16) = z;
      }
      fence_proxy_async_shared();
      mbar_arrive(&bars.full[s]);
    };
    fetch(0);
    publish(0);
    if (chunks > 1) fetch(1);
    for (int c = 0; c < chunks; ++c) {
      const int s = c % C_STAGES, ts = c % 2;
      const int i = t & 63;       // this thread's step: row of K K^T (t < 64) or of Q K^T
      wait(&bars.g_full, c);
      tc_fence_after();
      const uint32_t gaddr = tmem + (uint32_t(warp * 32) << 16) + C::COL_G;
      if (c >= 2) wait(&bars.tp_freed[ts], (c / 2) - 1);
      const float* gs = g_of(s);
      uint8_t* tp = smem + C::TP_OFF + ts * C::TP_BYTES;
      float* diag = reinterpret_cast<float*>(smem + C::A_OFF);
      float* off32 = diag + 6 * DIAG_BLK;
      float* nowhere = off32 + 32 * OFF_LD + lane * 8;
      // D_ij along the row, from the diagonal to the left, times beta_i in A's
      // rows; right of the diagonal d is 0 (what A's diagonal holds is not read)
      const float start = t < 64 ? b_of(s)[i] : 1.f;
      // A's row in fp32: lanes of a warp differ in which block a column is in,
      // and lanes that a store is not for have a place for it, so that no
      // branch splits the warp
      const int blk = i / 16;
      float* row_diag = diag + blk * DIAG_BLK + (i % 16) * DIAG_LD;
      float* row_odd = blk & 1 ? row_diag : nowhere;                                  // columns of block 1 or 3
      float* row_even = blk & 1 ? row_diag + (4 + blk / 2 - blk) * DIAG_BLK : row_diag;  // of block 0 or 2
      float d = 0.f, next = 0.f;
      // the first 32 rows end with column 31
      int j8 = warp & 1 ? CH - 8 : 24;
      uint32_t gr[8];
      tmem_ld_32x32b_x8(gaddr + j8, gr);
#pragma unroll 1
      for (; j8 >= 0; j8 -= 8) {
        const float4 glo = at4(gs + j8), ghi = at4(gs + j8 + 4);
        const float gg[8] = {glo.x, glo.y, glo.z, glo.w, ghi.x, ghi.y, ghi.z, ghi.w};
        float o[8];
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(gr[e]);
        if (j8 > 0) tmem_ld_32x32b_x8(gaddr + j8 - 8, gr);
#pragma unroll
        for (int e = 7; e >= 0; --e) {
          d = j8 + e == i ? start : d * next;
          next = gg[e];
          o[e] *= d;
        }
        if (t >= 64) {
          *reinterpret_cast<uint4*>(tp + 3 * PART + part_at(i, j8)) = take_part8(o);
          *reinterpret_cast<uint4*>(tp + 4 * PART + part_at(i, j8)) = take_part8(o);
        } else {
          float* at = warp == 1 && j8 < 32 ? off32 + (i - 32) * OFF_LD + j8
                                           : ((j8 / 16) & 1 ? row_odd : row_even) + (j8 % 16);
          *reinterpret_cast<float4*>(at) = make_float4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<float4*>(at + 4) = make_float4(o[4], o[5], o[6], o[7]);
        }
      }
      tc_fence_before();
      mbar_arrive(&bars.g_read);
      named_bar_sync(1, C_PREP);
      if (t < 64) {
        invert_block16(diag + (t / 16) * DIAG_BLK, t % 16);
      } else {
        // c_i (warp 2) and D_63,j (warp 3): products of the decays up to a step
        // and behind it, two steps per lane
        const float2 gg = *reinterpret_cast<const float2*>(gs + 2 * lane);
        float x = gg.x * gg.y;
        if (warp == 2) {
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const float y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x *= y;
          }
          float before = __shfl_up_sync(0xffffffffu, x, 1);
          if (lane == 0) before = 1.f;
          before *= gg.x;
          const float2 bb = *reinterpret_cast<const float2*>(b_of(s) + 2 * lane);
          *reinterpret_cast<float2*>(cum_of(ts) + 2 * lane) = make_float2(before, x);
          *reinterpret_cast<float2*>(nbc_of(ts) + 2 * lane) = make_float2(-bb.x * before, -bb.y * x);
        } else {
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const float y = __shfl_down_sync(0xffffffffu, x, o);
            if (lane + o < 32) x *= y;
          }
          x = __shfl_down_sync(0xffffffffu, x, 1);
          if (lane == 31) x = 1.f;
          *reinterpret_cast<float2*>(until_of(ts) + 2 * lane) = make_float2(x * gg.y, x);
        }
      }
      // halfway: the next chunk's tiles have had the time to land, and its
      // [K; Q] K^T is there when this chunk's T is done
      if (c + 1 < chunks) publish(c + 1);
      if (c + 2 < chunks) fetch(c + 2);
      named_bar_sync(1, C_PREP);
      // The rest of the inverse from its diagonal blocks: blocks of 16, then of
      // 32.  On the register form of the tensor instructions: at these sizes a
      // TMEM round trip would cost more than the products.
      if (warp < 2)
        join16(diag, tp, warp, lane);
      else
        store_diag_row(diag, tp, (t - 64) / 16, t % 16);
      named_bar_sync(1, C_PREP);
      join32(diag, off32, tp, (warp / 2) * 16, (warp % 2) * 16, lane);
      fence_proxy_async_shared();
      mbar_arrive(&bars.tp_full[ts]);
      named_bar_sync(1, C_PREP);   // before the next A goes over this one's
    }
  } else if (warp < 12) {
    // --------------------------------------------------------- the state rows
    more_registers<C_REGS_STATE>();
    const int h = (warp - 4) / 4;            // which half of the columns
    const int row = (warp % 4) * 32 + lane;  // TMEM lane, value row dv0 + row
    const uint32_t ta = tmem + (uint32_t((warp % 4) * 32) << 16);
    constexpr int NS = DK / 2;               // state columns of this thread
    // The warp's 32 rows of half the columns go through shared memory both ways,
    // so that neighbouring lanes read and write neighbouring 16 bytes (with a row
    // per lane the state's 64 KB took 3400 cycles to come, the first chunk's
    // copies waiting behind them, and 5900 to go).
    constexpr int X = NS / 4;                // 16-byte pieces of a row
    auto piece_of = [&](float4* part, int r, int x) { return part + r * X + (x ^ (r & (X - 1))); };
    float s[NS];
    if (src) {
      // over the second and third stage, which wait for s_ready
      float4* part = reinterpret_cast<float4*>(smem + C::KQ_BYTES) + (warp - 4) * 32 * X;
#pragma unroll
      for (int i = 0; i < X; ++i) {
        const int r = i * (32 / X) + lane / X, x = lane % X, at = (warp % 4) * 32 + r;
        cp_async_16(smem_u32(piece_of(part, r, x)), src + (size_t)(at < cols ? at : 0) * DK + h * NS + 4 * x,
                    at < cols ? 16 : 0);
      }
      cp_async_commit();
      cp_async_wait_all();
      __syncwarp();
#pragma unroll
      for (int i = 0; i < X; ++i) {
        const float4 x = *piece_of(part, lane, i);
        s[4 * i] = x.x; s[4 * i + 1] = x.y; s[4 * i + 2] = x.z; s[4 * i + 3] = x.w;
      }
      fence_proxy_async_shared();
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i) s[i] = unit && row == h * NS + i ? 1.f : 0.f;
    }
    const uint32_t s_col = ta + C::COL_S + h * (NS / 2);
    float r[32];
    auto beta_v = [&](int c) {               // r = beta V of chunk c
      const int st = c % C_STAGES;
      wait(&bars.full[st], c / C_STAGES);    // beta
      wait(&bars.v_loaded[c % 2], c / 2);
      const __nv_bfloat16* vt =
          reinterpret_cast<const __nv_bfloat16*>(smem + C::V_OFF + (c % 2) * C::V_BYTES) + h * 32 * 128 + row;
      const float* bs = b_of(st) + h * 32;
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = __bfloat162float(vt[j * 128]);
      // beta is 0 at steps of no sequence and masked ones, whatever V holds there
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 x = at4(bs + j);
        const float be[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = be[e] * r[j + e];
          r[j + e] = be[e] == 0.f || unit ? 0.f : y;
        }
      }
    };
    const size_t y_step = (size_t)p.Hv * p.Dv;
    __nv_bfloat16* out = p.y + ((first + h * 32) * p.Hv + hv) * p.Dv + dv0;
    auto yt_of = [&](int c) { return smem + C::V_OFF + (c % 2) * C::V_BYTES + h * 32 * 256; };
    uint32_t d[2][16];
    float co[16];
    // Turn c ends chunk c - 1 (its state, its y) and begins chunk c.
#pragma unroll 1
    for (int c = 0;; ++c) {
      if (c < chunks) beta_v(c);               // while the last chunk's Delta K runs
      // S <- c_63 S + Delta K, and its parts for the products
      float keep = 0.f;
      if (c > 0) {
        keep = cum_of((c - 1) % 2)[CH - 1];
        wait(&bars.d4_done, c - 1);
        tc_fence_after();
        tmem_ld_32x32b_x16(ta + C::COL_D + h * NS, d[0]);
      }
#pragma unroll
      for (int b = 0; b < NS / 16; ++b) {
        if (c > 0) {
          tmem_ld_wait();
          if (b + 1 < NS / 16) tmem_ld_32x32b_x16(ta + C::COL_D + h * NS + 16 * (b + 1), d[(b + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 16; j += 2)
            fma2(s[16 * b + j], s[16 * b + j + 1], keep, keep, s[16 * b + j], s[16 * b + j + 1],
                 __uint_as_float(d[b & 1][j]), __uint_as_float(d[b & 1][j + 1]));
        }
        if (c < chunks) {
          float x[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = s[16 * b + j];
          store_parts<3>({s_col + 8 * b, s_col + C::S_PART + 8 * b, s_col + 2 * C::S_PART + 8 * b}, x);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      // The last turn's y was written and read in V's buffer; the copy that fills
      // it next is issued once this arrival is there, and a barrier alone does
      // not order these accesses before a TMA write.
      fence_proxy_async_shared();
      mbar_arrive(&bars.s_ready);
      if (c > 0) {
        // Y = c Q S^T + P Delta of the last chunk, while this one's K S^T runs.
        // Steps are rows of y and value rows its columns: the tile is turned in
        // shared memory, so that y goes out 16 bytes a lane (2-byte stores
        // straight from the lanes took 2700 cycles of a chunk's 10000 with every
        // SM at work).  It lies over this chunk's V, which every thread has read
        // before s_ready.
        const int last = c - 1, ts = last % 2;
        wait(&bars.y_done, last);
        if (!partial) {
          const float* cs = cum_of(ts) + h * 32;
          tc_fence_after();
          load16(cs, co);
          tmem_ld_32x32b_x16(ta + C::COL_SQ + h * 32, d[0]);
          tmem_ld_32x32b_x16(ta + C::COL_Y + h * 32, d[1]);
          wait(&bars.s_ready, c);
          __nv_bfloat16* at = reinterpret_cast<__nv_bfloat16*>(yt_of(c)) + row;
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              at[j * 128] = __float2bfloat16_rn(__fmaf_rn(co[j], __uint_as_float(d[0][j]), __uint_as_float(d[1][j])));
            at += 16 * 128;
            if (b == 0) {
              load16(cs + 16, co);
              tmem_ld_32x32b_x16(ta + C::COL_SQ + h * 32 + 16, d[0]);
              tmem_ld_32x32b_x16(ta + C::COL_Y + h * 32 + 16, d[1]);
            }
          }
          tc_fence_before();
        }
        mbar_arrive(&bars.y_read);
        if (!partial) {
          named_bar_sync(2 + h, C_STATE / 2);
          const int rows = min(CH, len - last * CH) - h * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = (warp % 4) * 8 + 2 * i + lane / 16, x = lane % 16;
            const uint4 u = *reinterpret_cast<const uint4*>(yt_of(c) + rr * 256 + x * 16);
            if (rr < rows && x * 8 < cols) *reinterpret_cast<uint4*>(out + rr * y_step + x * 8) = u;
          }
          out += CH * y_step;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.tp_freed[ts]);
      }
      if (c == chunks) break;
      const int ts = c % 2;
      // R = beta V - beta c K S^T.  Coefficients come 16 at a time, ahead of the
      // stores that the compiler keeps loads behind.
      wait(&bars.tp_full[ts], c / 2);
      const float* us = until_of(ts) + h * 32;
      const float* nbc = nbc_of(ts) + h * 32;
      load16(nbc, co);
      wait(&bars.d1_done, c);
      tc_fence_after();
      tmem_ld_32x32b_x16(ta + C::COL_D + h * 32, d[0]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        tmem_ld_wait();
        if (b == 0) tmem_ld_32x32b_x16(ta + C::COL_D + h * 32 + 16, d[1]);
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const int jj = 16 * b + j;
          fma2(r[jj], r[jj + 1], co[j], co[j + 1], __uint_as_float(d[b][j]), __uint_as_float(d[b][j + 1]), r[jj],
               r[jj + 1]);
          x[j] = r[jj];
          x[j + 1] = r[jj + 1];
        }
        if (b == 0) load16(nbc + 16, co);
        store_parts<3>({ta + C::COL_R + h * 16 + 8 * b, ta + C::COL_R + 32 + h * 16 + 8 * b,
                        ta + C::COL_Y + h * 32 + 8 * b}, x);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars.r_ready);
      // Delta = R + (T - I) R, as it is (for y) and weighed for the state
      load16(us, co);
      wait(&bars.q_done, c);                 // S Q^T has read the state that the parts of Delta go over
      wait(&bars.d3_done, c);
      tc_fence_after();
      tmem_ld_32x32b_x16(ta + C::COL_D + h * 32, d[0]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        tmem_ld_wait();
        if (b == 0) tmem_ld_32x32b_x16(ta + C::COL_D + h * 32 + 16, d[1]);
        float x[16], w[16];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const int jj = 16 * b + j;
          fma2(x[j], x[j + 1], 1.f, 1.f, __uint_as_float(d[b][j]), __uint_as_float(d[b][j + 1]), r[jj], r[jj + 1]);
          fma2(w[j], w[j + 1], co[j], co[j + 1], x[j], x[j + 1], 0.f, 0.f);
        }
        if (b == 0) load16(us + 16, co);
        store_parts<3>({ta + C::COL_S + h * 16 + 8 * b, ta + C::COL_S + 32 + h * 16 + 8 * b,
                        ta + C::COL_S + 64 + h * 16 + 8 * b}, w);
        store_parts<2>({ta + C::COL_R + h * 16 + 8 * b, ta + C::COL_R + 32 + h * 16 + 8 * b}, x);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars.delta_ready);
    }
    if (dst) {
      // over the first two stages, which every product has read
      float4* part = reinterpret_cast<float4*>(smem) + (warp - 4) * 32 * X;
#pragma unroll
      for (int i = 0; i < X; ++i)
        *piece_of(part, lane, i) = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < X; ++i) {
        const int r = i * (32 / X) + lane / X, x = lane % X, at = (warp % 4) * 32 + r;
        if (at < cols) *reinterpret_cast<float4*>(dst + (size_t)at * DK + h * NS + 4 * x) = *piece_of(part, r, x);
      }
    }
  } else {
    // ----------------------------------------------------- loads and products
    fewer_registers<C_REGS_ISSUE>();
    // The whole warp walks along, one elected lane issues.  The chain from one
    // state to the next and what only has to be done beside it are issued by
    // two warps; a product that reads what the other's wrote, or writes what it
    // read, comes after a wait that covers it.
    constexpr uint32_t ID64 = make_idesc_bf16(128, 64);
    constexpr uint32_t IDK = make_idesc_bf16(128, DK) | kIdescBTransposed;
    if (warp == 12) {
      for (int c = 0; c < chunks; ++c) {
        const int ts = c % 2;
        const uint32_t kq = smem_base + (c % C_STAGES) * C::KQ_BYTES;
        const uint32_t tp = smem_base + C::TP_OFF + ts * C::TP_BYTES;
        wait(&bars.full[c % C_STAGES], c / C_STAGES);
        wait(&bars.s_ready, c);
        tc_fence_after();
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int a = 0; a < DK / 64; ++a)
            mma_bf16_ts_warp_x4<2>(tmem + C::COL_D, tmem + C::COL_S + part * C::S_PART + a * 32,
                                   make_sw128_desc(kq + a * C::ATOM), ID64, part < 2 || a > 0);
        tc_commit_warp(&bars.d1_done);
        wait(&bars.tp_full[ts], c / 2);
        wait(&bars.r_ready, c);
        tc_fence_after();
        // two parts of R with two of T, the third ones with the other's first
#pragma unroll
        for (int k = 0; k < CH / 16; ++k)
          mma_bf16_ts_warp(tmem + C::COL_D, tmem + C::col_r3(k), make_sw128_desc(tp + k * 32), ID64, k > 0);
        mma_bf16_ts_warp_x4<2>(tmem + C::COL_D, tmem + C::COL_R, make_sw128_desc(tp + 2 * PART), ID64, 1);
#pragma unroll
        for (int m = 3; m >= 0; --m)
          mma_bf16_ts_warp_x4<2>(tmem + C::COL_D, tmem + C::COL_R + (m & 1 ? 32 : 0),
                                 make_sw128_desc(tp + (m & 2 ? PART : 0)), ID64, 1);
        tc_commit_warp(&bars.d3_done);
        wait(&bars.delta_ready, c);
        // [K; Q] K^T of the next chunk has left the second half of these columns
        if (c + 1 < chunks) wait(&bars.g_read, c + 1);
        tc_fence_after();
#pragma unroll
        for (int part = 2; part >= 0; --part)
          mma_bf16_ts_warp_x4<128>(tmem + C::COL_D, tmem + C::COL_S + part * 32, make_sw128_mn_desc(kq, C::ATOM), IDK,
                                   part < 2);
        tc_commit_warp(&bars.d4_done);
      }
    } else if (warp == 14) {
      auto grams = [&](int c) {   // [K; Q] K^T
        const uint32_t kq = smem_base + (c % C_STAGES) * C::KQ_BYTES;
        wait(&bars.full[c % C_STAGES], c / C_STAGES);
#pragma unroll
        for (int a = 0; a < DK / 64; ++a)
          mma_bf16_ss_warp_x4(tmem + C::COL_G, make_sw128_desc(kq + a * C::ATOM), make_sw128_desc(kq + a * C::ATOM), ID64,
                              a > 0);
        tc_commit_warp(&bars.g_full);
      };
      grams(0);
      wait(&bars.g_read, 0);
      for (int c = 0; c < chunks; ++c) {
        const int ts = c % 2;
        const uint32_t kq = smem_base + (c % C_STAGES) * C::KQ_BYTES;
        const uint32_t tp = smem_base + C::TP_OFF + ts * C::TP_BYTES;
        wait(&bars.s_ready, c);
        // the last chunk's Delta K has been read, its second half is free until
        // this chunk's
        tc_fence_after();
        if (c + 1 < chunks) grams(c + 1);
        if (c > 0) wait(&bars.y_read, c - 1);
        tc_fence_after();
#pragma unroll
        for (int part = 1; part >= 0; --part)
#pragma unroll
          for (int a = 0; a < DK / 64; ++a)
            mma_bf16_ts_warp_x4<2>(tmem + C::COL_SQ, tmem + C::COL_S + part * C::S_PART + a * 32,
                                   make_sw128_desc(kq + 64 * 128 + a * C::ATOM), ID64, part < 1 || a > 0);
        tc_commit_warp(&bars.q_done);
        wait(&bars.delta_ready, c);
        tc_fence_after();
#pragma unroll
        for (int m = 2; m >= 0; --m)
          mma_bf16_ts_warp_x4<2>(tmem + C::COL_Y, tmem + C::COL_R + (m == 1 ? 32 : 0),
                                 make_sw128_desc(tp + (m == 2 ? 4 : 3) * PART), ID64, m < 2);
        tc_commit_warp(&bars.y_done);
        tc_commit_warp(&bars.tp_freed[ts]);
      }
      // the last arrivals land before the CTA gives its memory back (the other
      // commits' were waited for by the state's threads)
      for (int c = max(0, chunks - 2); c < chunks; ++c) wait(&bars.tp_freed[c % 2], c / 2);
    } else if (warp == 13 && lane == 0) {
      // loads, on a thread of their own: issuing a chunk's five takes about as
      // long (2000 cycles) as a round of products
      auto load_v = [&](int c) {
        uint64_t* bar = &bars.v_loaded[c % 2];
        mbar_arrive_expect_tx(bar, C::V_BYTES);
        tma_load_2d(smem + C::V_OFF + (c % 2) * C::V_BYTES, &tm_v, bar, hv * p.Dv + dv0, int(first) + c * CH);
      };
      auto load_kq = [&](int c) {
        uint8_t* kq = smem + (c % C_STAGES) * C::KQ_BYTES;
        uint64_t* bar = &bars.loaded[c % C_STAGES];
        const int tok = int(first) + c * CH;
        mbar_arrive_expect_tx(bar, C::KQ_BYTES);
        for (int a = 0; a < DK / 64; ++a) {
          tma_load_2d(kq + a * C::ATOM, &tm_k, bar, hk * DK + a * 64, tok);
          tma_load_2d(kq + a * C::ATOM + 64 * 128, &tm_q, bar, hk * DK + a * 64, tok);
        }
      };
      load_kq(0);
      load_v(0);
      for (int c = 1; c < chunks; ++c) {
        // Chunk c - 3 is done with the stage: its products are complete (the next
        // state came after them).  So is V's buffer of chunk c - 3, over which
        // the y of chunk c - 4 was turned: it takes chunk c - 1.  Every phase is
        // waited for in turn: a parity alone does not tell phase 1 from none.  The
        // first state came through the stages of chunks 1 and 2.
        if (c == 1) wait(&bars.s_ready, 0);
        if (c >= C_STAGES) {
          wait(&bars.s_ready, c - C_STAGES + 1);
          load_v(c - 1);
        }
        load_kq(c);
        if (c == 1) load_v(1);
      }
      if (chunks >= C_STAGES) {
        wait(&bars.s_ready, chunks - C_STAGES + 1);
        load_v(chunks - 1);
      }
      // whatever went wrong elsewhere, no copy is in flight when the CTA leaves
      for (int c = max(0, chunks - C_STAGES); c < chunks; ++c)
        mbar_wait(&bars.loaded[c % C_STAGES], (c / C_STAGES) & 1);
      for (int c = max(0, chunks - 2); c < chunks; ++c) mbar_wait(&bars.v_loaded[c % 2], (c / 2) & 1);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// Pieces of a sequence (lengths of packed ones are known on the device only:
// their mean is taken, so a long one beside many short ones is not cut).  In units
// of a chunk's time (6.1 us): whole, L; in n pieces, two launches of L / n chunks that
// are 1.06 long with every SM at work, 6 for starting two launches more and 0.6 for a
// step of the chain.  Measured, us whole and cut: 48 heads 781 / 601 at 8192 steps, 398 /
// 329 at 4096 and 204 / 181 at 2048 (3 pieces; 107 / 112 at 1000, left whole), 16 heads
// 773 / 323 at 8192 and 200 / 112 at 2048 (6), 4 heads 770 / 169 (16) and 199 / 95 (10 or
// 16), 8 heads of 64 x 64 687 / 180 and 177 / 75 (10).
inline int pieces(long long heads, int tiles, long long chunks, int sms) {
  int best = 1;
  double least = 0.95 * double(chunks);
  for (int n = 3; n <= MAX_PIECES; ++n) {
    if (heads * (tiles * (n - 1) + n - 2) > sms) break;
    const double cost = 2.12 * double((chunks + n - 1) / n) + 6.0 + 0.6 * (n - 2);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

inline size_t split_layout(Split* sp, uint8_t* base, size_t heads, int Dv, int Dk) {
  const size_t state = (size_t)Dv * Dk * 4, square = (size_t)Dk * Dk * 4;
  sp->start = reinterpret_cast<float*>(base);
  sp->add = reinterpret_cast<float*>(base + heads * (sp->n - 1) * state);
  sp->map = reinterpret_cast<float*>(base + heads * (2 * sp->n - 3) * state);
  return sp->n == 1 ? 0 : heads * ((2 * sp->n - 3) * state + (sp->n - 2) * square);
}

inline int split_of(int B, int T, bool packed, int Hv, int Dv, int sms) {
  if (B < 1) return 1;
  const long long steps = packed ? T / B : T;
  return pieces((long long)B * Hv, (Dv + 127) / 128, (steps + CH - 1) / CH, sms);
}

template <int DK>
int launch_chunked(const RuleParams& p, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const int tiles = (p.Dv + 127) / 128;
  const long long heads = (long long)p.B * p.Hv;
  if (heads * tiles > 0x7fffffffll || (!p.cu && (long long)p.B * p.T > 0x7fffffffll)) return DFL_ERR_BAD_SHAPE;
  int dev, sms;
  int st = host::current_device(&dev, &sms);
  if (st != DFL_OK) return st;
  Split sp;
  sp.n = split_of(p.B, p.T, p.cu != nullptr, p.Hv, p.Dv, sms);
  sp.last = 0;
  sp.jobs = sp.n == 1 ? tiles : tiles * (sp.n - 1) + sp.n - 2;
  const size_t need = split_layout(&sp, reinterpret_cast<uint8_t*>(workspace), heads, p.Dv, DK);
  if (need > 0 && (!workspace || workspace_bytes < need)) return DFL_ERR_WORKSPACE;
  if (need > 0 && !host::aligned(workspace, 16)) return DFL_ERR_MISALIGNED;
  st = host::ensure_smem(gdn_rule_chunked<DK>, CCfg<DK>::SMEM_BYTES, dev, done);
  if (st != DFL_OK) return st;
  static std::atomic<uint64_t> chain_done{0};
  st = host::ensure_smem(gdn_rule_chain<DK>, chain_smem<DK>(), dev, chain_done);
  if (st != DFL_OK) return st;
  const uint64_t tokens = p.cu ? uint64_t(p.T) : uint64_t(p.B) * p.T;
  CUtensorMap tm_q, tm_k, tm_v;
  if (tokens > 0) {
    const uint64_t wk = uint64_t(p.Hk) * DK, wv = uint64_t(p.Hv) * p.Dv;
    st = host::make_tmap_2d(&tm_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.q, wk, tokens, uint64_t(p.ldq) * 2, 64, CH,
                            CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != DFL_OK) return st;
    st = host::make_tmap_2d(&tm_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.k, wk, tokens, uint64_t(p.ldk) * 2, 64, CH,
                            CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != DFL_OK) return st;
    st = host::make_tmap_2d(&tm_v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.v, wv, tokens, uint64_t(p.ldv) * 2, 128, CH,
                            CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st != DFL_OK) return st;
  } else {
    std::memset(&tm_q, 0, sizeof(tm_q));   // no step, no load
    tm_k = tm_v = tm_q;
  }
  gdn_rule_chunked<DK><<<int(heads * sp.jobs), C_THREADS, CCfg<DK>::SMEM_BYTES, stream>>>(tm_q, tm_k, tm_v, p, sp);
  st = host::launch_status();
  if (st != DFL_OK || sp.n == 1) return st;
  gdn_rule_chain<DK><<<int(heads * (p.Dv / CHAIN_ROWS)), 2 * DK, chain_smem<DK>(), stream>>>(sp, p.Dv);
  st = host::launch_status();
  if (st != DFL_OK) return st;
  sp.last = 1;
  sp.jobs = tiles * (sp.n - 1);
  gdn_rule_chunked<DK><<<int(heads * sp.jobs), C_THREADS, CCfg<DK>::SMEM_BYTES, stream>>>(tm_q, tm_k, tm_v, p, sp);
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

extern "C" int dfl_gdn_rule_chunked(const uint16_t* q, int ldq, const uint16_t* k, int ldk, const uint16_t* v,
                                    int ldv, const float* g, const float* beta, const uint8_t* mask,
                                    const int32_t* cu_seqlens, const float* state_in, float* state_out,
                                    uint16_t* y, int zero_gaps, int B, int T, int Hv, int Hk, int Dv, int Dk,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dfl;
  gdnr::RuleParams p;
  bool done;
  const int st = gdnr::rule_params(q, ldq, k, ldk, v, ldv, g, 0, beta, mask, cu_seqlens, state_in, state_out, y,
                                   zero_gaps, B, T, Hv, Hk, Dv, Dk, &p, &done);
  if (st != DFL_OK || done) return st;
  if (Dk != 64 && Dk != 128) return DFL_ERR_BAD_SHAPE;
  // 16-byte copies: tokens and heads on 16-byte borders
  if (ldq % 8 != 0 || ldk % 8 != 0 || ldv % 8 != 0 || !host::aligned(q, 16) || !host::aligned(k, 16) ||
      !host::aligned(v, 16))
    return DFL_ERR_MISALIGNED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return Dk == 64 ? gdnr::launch_chunked<64>(p, workspace, workspace_bytes, s)
                  : gdnr::launch_chunked<128>(p, workspace, workspace_bytes, s);
}

extern "C" size_t dfl_gdn_rule_workspace_bytes(int B, int T, int packed, int Hv, int Dv, int Dk, int* status) {
  using namespace dfl;
  int dummy;
  int* st = status ? status : &dummy;
  if (B < 0 || T < 0 || Hv < 1 || Dv < 32 || Dv % 32 != 0 || (Dk != 64 && Dk != 128)) {
    *st = DFL_ERR_BAD_SHAPE;
    return 0;
  }
  int dev, sms;
  *st = host::current_device(&dev, &sms);
  if (*st != DFL_OK) return 0;
  gdnr::Split sp;
  sp.n = gdnr::split_of(B, T, packed != 0, Hv, Dv, sms);
  return gdnr::split_layout(&sp, nullptr, (size_t)B * Hv, Dv, Dk);
}
