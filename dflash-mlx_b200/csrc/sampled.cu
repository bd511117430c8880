// Verification of drafted tokens against the target's probabilities (sm_100a).
//
// For request b with temperature z, drafts x_1 .. x_n (n = draft_lens[b]), row i
// of the target's logits after the i-th token of the block and, where the draft
// model's logits are given, row i of those for the draft x_{i+1}:
//     p_i = softmax(logits_i / z) without the suppressed ids,
//     q_i = softmax(draft_i / z), or all on x_{i+1} (greedy drafts),
//     draft i is accepted while u_i q_i(x_{i+1}) < p_i(x_{i+1});  a = accepted,
//     next token ~ max(p_a - q_a, 0) when a < n, else ~ p_n, by inverse
//     cumulative sum in id order: the first id whose sum exceeds sample_u x total.
// The committed tokens are then distributed as samples of the target alone.
// z = 0 (or below, or NaN) is greedy: p_i is all on the largest logit's id.
//
// Three to five launches, each after the first started early.  mask_kernel packs
// the suppress mask into bits, if there is one.  rows_kernel reads every row once
// (the one pass that is bound by HBM): maximum, its id and sum of exponentials
// of each segment, in 32 bits.
// decide_kernel joins a request's segments and accepts.  Where the next token
// comes from a difference of two softmaxes, norm_kernel adds the two rows'
// exponentials again in 64 bits.  pick_kernel adds the weights of that one
// row's segments in 64 bits, and the last CTA of a request finds the segment and
// the id.  The 64 bits are for the id: with 2^18 ids a weight is 2^-18 of the
// total, and a sum in 32 bits would move a border by a sizeable part of it.
//
// A logit that is NaN or -inf has probability 0; rows with +inf spread over
// those ids.  A row that has nothing left gives token -1.
//
// Replaces, for sampled decoding, the greedy tail of dflash_mlx/engine/
// spec_epoch.py:2067-2072,2129 (greedy_tokens_with_mask engine/sampling.py:47-55
// and match_acceptance_length engine/acceptance.py:9-16).

namespace dfl {
namespace smp {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCK = 256;    // tokens of a block
constexpr int PICK_SEG = 512;     // ids of a segment of the picked row, a warp's

struct Params {
  const void* logits;    // [B, T] rows of V
  const void* draft;     // [B, T - 1] rows of V, or null
  const int32_t* ids;    // [B, T]
  const float* accept_u; // [B, T - 1]
  const float* sample_u; // [B]
  const float* temperature;  // [B]
  const int32_t* lens;   // [B] or null
  const uint8_t* suppress;   // [V] or null
  int32_t* accepted;     // [B]
  int32_t* token;        // [B]
  float* draft_prob;     // [B, T - 1]
  long long ld, ldd;     // elements from one row to the next
  long long bs, bsd;     // elements from one request to the next
  int B, T, V;
  int segs, seg;         // segments of a row and their length (rows_kernel)
  int psegs;             // segments of PICK_SEG ids (pick_kernel)
  int words;             // of the mask's bits
  int group;             // segments of a warp (norm_kernel, pick_kernel)
  // workspace
  uint32_t* bits;        // [words]
  float2* part;          // [B * T + B * (T - 1)][segs] (maximum, sum)
  int* part_id;          // [B * T][segs] lowest id of the maximum
  double* zsum;          // [2][B][CTAs of norm_kernel]
  double* wsum;          // [B][psegs]
  struct Chosen* chosen; // [B]
  int* ticket;           // [B]
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// 0 for greedy, else the temperature kept where 1 / z and FLT_MAX / z are finite.
__device__ __forceinline__ float clean_temperature(float z) {
  return z > 0.f ? fminf(fmaxf(z, 1e-30f), 1e30f) : 0.f;
}

__device__ __forceinline__ int draft_len(const Params& p, int b) {
  if (!p.lens) return p.T - 1;
  const int n = p.lens[b];
  const int c = min(max(n, 0), p.T - 1);
  if (c != n && threadIdx.x == 0) atomicExch(&g_device_error, kDevBadInput);
  return c;
}

template <typename T>
__device__ __forceinline__ const T* target_row(const Params& p, int b, int i) {
  return reinterpret_cast<const T*>(p.logits) + ((size_t)b * p.bs + (size_t)i * p.ld);
}

template <typename T>
__device__ __forceinline__ const T* draft_row(const Params& p, int b, int i) {
  return reinterpret_cast<const T*>(p.draft) + ((size_t)b * p.bsd + (size_t)i * p.ldd);
}

// (maximum, lowest id of it, sum of exp((x - maximum) / z)) of some ids; an
// empty set is (-inf, INT_MAX, 0).
struct Stat {
  float m, s;
  int id;
};

__device__ __forceinline__ float exp_scaled(float d, float c) {
  // d <= 0; NaN (a NaN logit) and -inf become -FLT_MAX: exp gives 0
  return exp2f(fmaxf(d, -FLT_MAX) * c);
}

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  r.id = a.m > b.m ? a.id : (b.m > a.m ? b.id : min(a.id, b.id));
  // a part that holds the maximum keeps its sum; the other one is scaled (equal
  // infinities would give NaN as a difference)
  r.s = (a.m == r.m ? a.s : a.s * exp_scaled(a.m - r.m, c)) + (b.m == r.m ? b.s : b.s * exp_scaled(b.m - r.m, c));
  return r;
}

__device__ __forceinline__ Stat warp_join(Stat a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.id = __shfl_xor_sync(0xffffffffu, a.id, o);
    a = join(a, b, c);
  }
  return a;
}

template <typename T>
__device__ __forceinline__ void take(Stat& a, float x, int id, float c) {
  if (x > a.m) {
    a.s = a.m == -INFINITY ? 0.f : (x == INFINITY ? 0.f : a.s * exp_scaled(a.m - x, c));
    a.m = x;
    a.id = id;
  }
  // at +inf only the ids that hold it count (inf - inf is NaN: 0)
  a.s += x == INFINITY ? 1.f : exp_scaled(x - a.m, c);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of logits: as floats, their largest (NaN only if all are), and -inf
// put over those with a bit in `off`.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float top(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ void hide(uint4& u, uint32_t off) {
    if (off & 1u) u.x = 0xff800000u;
    if (off & 2u) u.y = 0xff800000u;
    if (off & 4u) u.z = 0xff800000u;
    if (off & 8u) u.w = 0xff800000u;
  }
};

template <uint32_t NEG_INF>
__device__ __forceinline__ void hide16(uint4& u, uint32_t off) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((off >> (2 * i)) & 1u) w[i] = (w[i] & 0xffff0000u) | NEG_INF;
    if ((off >> (2 * i + 1)) & 1u) w[i] = (w[i] & 0xffffu) | (NEG_INF << 16);
  }
  u = make_uint4(w[0], w[1], w[2], w[3]);
}

template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float top(const uint4& u) {
    const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ void hide(uint4& u, uint32_t off) { hide16<0xff80u>(u, off); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const __half2* w = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
  static __device__ __forceinline__ float top(const uint4& u) {
    const __half2* w = reinterpret_cast<const __half2*>(&u);
    const float2 m = __half22float2(__hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ void hide(uint4& u, uint32_t off) { hide16<0xfc00u>(u, off); }
};

constexpr int MAX_SEG = 65536;

// One bit per id, set where it is suppressed, a word per thread; 16 mask bytes at
// a time where they lie on 16-byte borders.  Packed once per call: in every
// row's pass the bytes would cost half of the row's own traffic, and packing
// them there 2.5 instructions an id (measured).
__global__ void __launch_bounds__(THREADS) mask_kernel(const Params p) {
  griddep_launch_dependents();
  const uint8_t* sup = p.suppress;
  const bool wide = (reinterpret_cast<uintptr_t>(sup) & 15) == 0;
  const int i = blockIdx.x * THREADS + threadIdx.x;
  if (i >= p.words) return;
  uint32_t r = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int v = 32 * i + 16 * h;
    if (wide && v + 16 <= p.V) {
      const uint4 u = *reinterpret_cast<const uint4*>(sup + v);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      // a byte each to 0 or 1, then bits 0, 8, 16, 24 side by side at the top
      for (int j = 0; j < 4; ++j) r |= ((__vsetne4(w[j], 0) * 0x10204080u) >> 28) << (16 * h + 4 * j);
    } else {
      for (int j = 0; j < 16 && v + j < p.V; ++j) r |= uint32_t(sup[v + j] != 0) << (16 * h + j);
    }
  }
  p.bits[i] = r;   // two words behind the last id are read with it: 0
}

// Segment blockIdx.x of row blockIdx.y (target rows, then draft rows).
//
// Per id: widen, half a packed maximum, one FMA for (x - m) c with c = log2(e) / z,
// ex2, add.  m c is rounded once per maximum, a common factor of all terms that
// is taken out again at the end.  The quick loop moves the maximum at most
// once in U vectors; a thread that met NaN or +inf, or nothing above the
// lowest value but that, goes over its ids again one by one; one that met only
// -inf does not.  1488 bf16 rows of 248,320
// ids (739 MB): 158 us, 72% of the measured copy rate, bound by the issue of
// its 5 instructions an id beside the loads.
template <typename T>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Params p) {
  __shared__ Stat sh[WARPS];
  constexpr int N = Vec<T>::N, U = 4;
  griddep_launch_dependents();
  const int row = blockIdx.y;
  const bool is_draft = row >= p.B * p.T;
  const int r = is_draft ? row - p.B * p.T : row;
  const int per = is_draft ? p.T - 1 : p.T;
  const int b = r / per, i = r - b * per;
  const int n = draft_len(p, b);
  if (row == 0 && blockIdx.x == 0)
    for (int x = threadIdx.x; x < p.B; x += THREADS) p.ticket[x] = 0;
  if (is_draft ? i >= n : i > n) return;  // a row of no draft
  const float z = clean_temperature(p.temperature[b]);
  if (is_draft && z == 0.f) return;
  const float c = z == 0.f ? 1.f : 1.44269504f / z;
  const T* x = is_draft ? draft_row<T>(p, b, i) : target_row<T>(p, b, i);
  const bool sup = !is_draft && p.suppress != nullptr;
  const uint32_t* bits = p.bits;
  const int v0 = blockIdx.x * p.seg, v1 = min(p.V, v0 + p.seg);
  auto hidden = [&](int v) { return sup && ((bits[v / 32] >> (v & 31)) & 1u); };
  // ids up to the first 16-byte border one by one, then vectors, then the rest
  const int head = min(int((16 - (reinterpret_cast<uintptr_t>(x + v0) & 15)) & 15) / int(sizeof(T)), v1 - v0);
  const int vecs = (v1 - v0 - head) / N;
  const int body = v0 + head;
  Stat a{-INFINITY, 0.f, 0x7fffffff};
  // mc stays above -inf: -inf, and the lowest value where c > 1, add 0 and not NaN
  float mc = -FLT_MAX;
  float part[U] = {};        // the sum, in parts that do not wait for one another
  auto raise = [&](float top) {
    const float was = mc;
    a.m = top;
    mc = fmaxf(a.m * c, -FLT_MAX);
    const float f = ex2(was - mc);
    a.s *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) part[u] *= f;
  };
  // the next vectors are on their way while these are worked on
  const uint4* src = reinterpret_cast<const uint4*>(x + body);
  uint4 raw[U], ahead[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (int(threadIdx.x) + u * THREADS < vecs) ahead[u] = __ldg(src + threadIdx.x + u * THREADS);
  if (sup) griddep_wait();   // the mask's bits
  for (int k0 = threadIdx.x; k0 < vecs; k0 += THREADS * U) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * THREADS;
      raw[u] = ahead[u];
      if (k + U * THREADS < vecs) ahead[u] = __ldg(src + k + U * THREADS);
      if (k < vecs) {
        if (sup) {
          const int o = body + k * N;
          const uint32_t off = __funnelshift_r(bits[o / 32], bits[o / 32 + 1], o & 31) & ((1u << N) - 1u);
          if (off) Vec<T>::hide(raw[u], off);
        }
      } else {
        Vec<T>::hide(raw[u], (1u << N) - 1u);
      }
      top = fmaxf(top, Vec<T>::top(raw[u]));
    }
    if (top > a.m) {
      raise(top);
      a.id = 0;        // which one it is, a greedy row finds below
      if (z == 0.f) {
        a.id = 0x7fffffff;
#pragma unroll
        for (int u = U - 1; u >= 0; --u) {
          float f[N];
          Vec<T>::get(raw[u], f);
#pragma unroll
          for (int j = N - 1; j >= 0; --j)
            if (f[j] == top) a.id = body + (k0 + u * THREADS) * N + j;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[N];
      Vec<T>::get(raw[u], f);
#pragma unroll
      for (int j = 0; j < N; ++j) part[u] += ex2(__fmaf_rn(f[j], c, -mc));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) a.s += part[u];
  // the ragged ends, taken by the first threads
  const int tail = body + vecs * N;
  const bool in_head = threadIdx.x < head, in_tail = tail + int(threadIdx.x) < v1;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (!(e ? in_tail : in_head)) continue;
    const int v = (e ? tail : v0) + int(threadIdx.x);
    const float f = hidden(v) ? -INFINITY : to_f<T>(x[v]);
    if (f > a.m) {
      raise(f);
      a.id = v;
    } else if (f == a.m) {
      a.id = min(a.id, v);
    }
    a.s += ex2(__fmaf_rn(f, c, -mc));
  }
  const bool nothing = a.m == -INFINITY && a.s == 0.f;   // only -inf; NaN would be in the sum
  // the rounding of m c comes out of the sum: 2^d to second order
  const float d = float(fma(-double(a.m), double(c), double(mc))) * 0.693147181f;
  a.s = __fmaf_rn(a.s, __fmaf_rn(0.5f * d, d, d), a.s);
  if (nothing) {
    a = Stat{-INFINITY, 0.f, 0x7fffffff};
  } else if (!(a.s > 0.f && fabsf(d) < 1e-3f) || a.id == 0x7fffffff) {
    a = Stat{-INFINITY, 0.f, 0x7fffffff};
    if (in_head) {
      const int v = v0 + int(threadIdx.x);
      take<T>(a, hidden(v) ? -INFINITY : to_f<T>(x[v]), v, c);
    }
    for (int k = threadIdx.x; k < vecs; k += THREADS)
      for (int j = 0; j < N; ++j) {
        const int v = body + k * N + j;
        take<T>(a, hidden(v) ? -INFINITY : to_f<T>(x[v]), v, c);
      }
    if (in_tail) {
      const int v = tail + int(threadIdx.x);
      take<T>(a, hidden(v) ? -INFINITY : to_f<T>(x[v]), v, c);
    }
  }
  a = warp_join(a, c);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = threadIdx.x < WARPS ? sh[threadIdx.x] : Stat{-INFINITY, 0.f, 0x7fffffff};
    a = warp_join(a, c);
    if (threadIdx.x == 0) {
      p.part[(size_t)row * p.segs + blockIdx.x] = make_float2(a.m, a.s);
      if (!is_draft) p.part_id[(size_t)row * p.segs + blockIdx.x] = a.id;
    }
  }
}

// The whole row's statistics from its segments, in every lane of the warp;
// the sum of exponentials relative to the maximum in 64 bits.
__device__ __forceinline__ void row_stat(const Params& p, int row, bool with_id, float c, float* m, double* s,
                                         int* id) {
  const int lane = threadIdx.x & 31;
  float mx = -INFINITY;
  int at = 0x7fffffff;
  for (int g = lane; g < p.segs; g += 32) {
    const float x = p.part[(size_t)row * p.segs + g].x;
    const int i = with_id ? p.part_id[(size_t)row * p.segs + g] : 0;
    if (x > mx) {
      mx = x;
      at = i;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (om > mx || (om == mx && oa < at)) {
      mx = om;
      at = oa;
    }
  }
  double sum = 0.0;
  for (int g = lane; g < p.segs; g += 32) {
    const float2 x = p.part[(size_t)row * p.segs + g];
    sum += x.x == mx ? (double)x.y : (double)x.y * (double)exp_scaled(x.x - mx, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  *m = mx;
  *s = sum;
  *id = at;
}

// exp((x - m) / z) in 64 bits; 0 for NaN and -inf, 1 for +inf under a +inf maximum.
__device__ __forceinline__ double weight(float x, float m, double inv_z) {
  if (x == m) return 1.0;
  const double d = (double)x - (double)m;
  return d < 0.0 ? exp(d * inv_z) : 0.0;   // NaN compares false; -inf gives exp(-inf) = 0
}

// The same for many ids: 2^t, t = (x - m) c with c = log2(e) / z, as 2^e T[i] 2^r with
// t = e + i / 256 + r, |r| <= 2^-9: the 256 powers of 2^(1/256) from a table in shared
// memory, 2^r by its Taylor series to r^3 (the next term is 1.4e-13 of the
// result).  10 operations in 64 bits; the sums of a row then err by less than
// 1e-13 of their total, where exponentials in 32 bits would leave 1e-9 and with
// 2^18 ids move one border in some thousands over a uniform.
constexpr int POWERS = 256;

__device__ __forceinline__ void fill_powers(double* table) {
  for (int i = threadIdx.x; i < POWERS; i += THREADS) table[i] = exp2(double(i) / POWERS);
}

__device__ __forceinline__ double weight_table(float x, float m, double c, const double* table) {
  const double t = ((double)x - (double)m) * c;
  const double big = 6755399441055744.0 / POWERS;       // 1.5 * 2^52: t rounds to a multiple of 2^-8
  const double s = t + big;
  const int k = __double2loint(s);
  const double r = t - (s - big);
  constexpr double l1 = 0.69314718055994530942, l2 = l1 * l1 / 2.0, l3 = l1 * l1 * l1 / 6.0;   // ln 2
  const double p = fma(fma(fma(l3, r, l2), r, l1), r, 1.0);
  const double w = table[k & (POWERS - 1)] * p;
  const double v = __hiloint2double(__double2hiint(w) + ((k >> 8) << 20), __double2loint(w));
  if (x == m) return 1.0;
  return t > -1000.0 ? v : 0.0;                          // NaN compares false
}

// A lane's 16 ids of a segment of PICK_SEG: N at a time next to each other (16
// bytes), the lanes side by side.
template <typename T>
__device__ __forceinline__ int lane_id(int j) {
  constexpr int N = Vec<T>::N;
  return (j / N) * 32 * N + int(threadIdx.x & 31) * N + j % N;
}

// Their logits, -inf behind the vocabulary or where suppressed; every load is
// issued before the first is waited for.
template <typename T>
__device__ __forceinline__ void load_ids(const T* row, const uint32_t* bits, int seg, int V, float (&x)[16]) {
  constexpr int N = Vec<T>::N;
  const int v0 = seg * PICK_SEG;
  uint32_t off[16 / N];
  if (v0 + PICK_SEG <= V && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    uint4 u[16 / N];
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      const int v = v0 + lane_id<T>(i * N);
      u[i] = __ldg(reinterpret_cast<const uint4*>(row + v));
      off[i] = bits ? bits[v / 32] >> (v & 31) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      float f[N];
      Vec<T>::get(u[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) x[i * N + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      off[i] = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int v = v0 + lane_id<T>(i * N + j), at = min(v, V - 1);
        x[i * N + j] = to_f<T>(row[at]);
        if (v >= V || (bits && ((bits[at / 32] >> (at & 31)) & 1u))) off[i] |= 1u << j;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if ((off[j / N] >> (j % N)) & 1u) x[j] = -INFINITY;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ double block_sum(double x, double* sh) {
  x = warp_sum(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) r += sh[w];
  return r;
}

// Exclusive sum over the threads before this one, added in a fixed order.
__device__ __forceinline__ double before_me(double x, double* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double run = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = run;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < warp; ++w) base += sh[w];
  const double prev = __shfl_up_sync(0xffffffffu, run, 1);
  return lane == 0 ? base : base + prev;
}

// What a request's next token is drawn from, as decide_kernel leaves it.
struct Chosen {
  int row;        // accepted drafts
  float mp, mq;   // maxima of the target's and of the draft's row (-inf: empty, or not used)
};

// Accept: a CTA per request, a warp per draft.
constexpr int DECIDE_WARPS = 16;

template <typename T>
__global__ void __launch_bounds__(32 * DECIDE_WARPS) decide_kernel(const Params p) {
  __shared__ int first_bad;
  griddep_launch_dependents();
  griddep_wait();
  const int b = blockIdx.x;
  const int n = draft_len(p, b);
  const float z = clean_temperature(p.temperature[b]);
  const float c = z == 0.f ? 1.f : 1.44269504f / z;
  const double inv_z = z == 0.f ? 0.0 : 1.0 / (double)z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) first_bad = n;
  __syncthreads();
  for (int i = warp; i < p.T - 1; i += DECIDE_WARPS) {
    double px = 0.0, qx = 1.0;
    if (i < n) {
      const int x = p.ids[(size_t)b * p.T + i + 1];
      const bool in = x >= 0 && x < p.V;
      const int at = in ? x : 0;
      const bool hidden = !in || (p.suppress && p.suppress[at]);
      const float lx = to_f<T>(target_row<T>(p, b, i)[at]);
      const float dx = p.draft ? to_f<T>(draft_row<T>(p, b, i)[at]) : 0.f;
      float m;
      double s;
      int id;
      row_stat(p, b * p.T + i, true, c, &m, &s, &id);
      if (m > -INFINITY && !hidden) px = z == 0.f ? (x == id ? 1.0 : 0.0) : weight(lx, m, inv_z) / s;
      if (p.draft && z != 0.f) {
        row_stat(p, p.B * p.T + b * (p.T - 1) + i, false, c, &m, &s, &id);
        qx = m > -INFINITY && in ? weight(dx, m, inv_z) / s : 0.0;
      }
      if (lane == 0) {
        const double u = p.accept_u[(size_t)b * (p.T - 1) + i];
        if (!(u * qx < px)) atomicMin(&first_bad, i);
      }
    }
    if (lane == 0) p.draft_prob[(size_t)b * (p.T - 1) + i] = float(px);
  }
  __syncthreads();
  if (warp != 0) return;
  const int a = first_bad;
  Chosen ch{a, -INFINITY, -INFINITY};
  double s;
  int id, unused;
  row_stat(p, b * p.T + a, true, c, &ch.mp, &s, &id);
  if (p.draft && a < n && z != 0.f) row_stat(p, p.B * p.T + b * (p.T - 1) + a, false, c, &ch.mq, &s, &unused);
  if (lane == 0) {
    p.accepted[b] = a;
    p.chosen[b] = ch;
    if (z == 0.f) p.token[b] = ch.mp > -INFINITY ? id : -1;
  }
}

// The 64-bit sums of segment blockIdx.x of the two rows whose difference a
// request draws from.  Bound by 64-bit arithmetic (a dozen operations an
// exponential): 48 requests of 248,320 ids 34 us.
template <typename T>
__global__ void __launch_bounds__(THREADS) norm_kernel(const Params p) {
  __shared__ double sh[WARPS];
  __shared__ double powers[POWERS];
  griddep_launch_dependents();
  fill_powers(powers);
  griddep_wait();
  __syncthreads();
  const int b = blockIdx.y;
  const int n = draft_len(p, b);
  const float z = clean_temperature(p.temperature[b]);
  const Chosen ch = p.chosen[b];
  if (!(ch.row < n && z != 0.f)) return;
  const T* lp = target_row<T>(p, b, ch.row);
  const T* lq = draft_row<T>(p, b, ch.row);
  const double c64 = 1.44269504088896340736 / (double)z;   // log2(e) / z
  double sp = 0.0, sq = 0.0;
  for (int g = 0; g < p.group; ++g) {
    const int seg = (blockIdx.x * p.group + g) * WARPS + int(threadIdx.x >> 5);
    if (seg >= p.psegs) break;
    float x[16], y[16];
    load_ids<T>(lp, p.suppress ? p.bits : nullptr, seg, p.V, x);
    load_ids<T>(lq, nullptr, seg, p.V, y);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      sp += weight_table(x[j], ch.mp, c64, powers);
      sq += weight_table(y[j], ch.mq, c64, powers);
    }
  }
  if (!(ch.mp > -INFINITY)) sp = 0.0;   // rows with nothing in them
  if (!(ch.mq > -INFINITY)) sq = 0.0;
  sp = block_sum(sp, sh);
  sq = block_sum(sq, sh);
  if (threadIdx.x == 0) {
    p.zsum[(size_t)b * gridDim.x + blockIdx.x] = sp;
    p.zsum[(size_t)(p.B + b) * gridDim.x + blockIdx.x] = sq;
  }
}

// What pick_kernel draws from: the target's row, the draft's row and id.
template <typename T>
struct Pick {
  const T* lp;
  const T* lq;     // null: no draft row to take away
  float mp, mq;
  double c64, ip, iq;    // log2(e) / z, 1 / sums
  const double* powers;
  int hot;         // id that a greedy draft takes away whole, or -1
  // weight of id v, target logit x (-inf: hidden) and draft logit y, left after
  // the draft.  The two products are rounded alike, not fused into the
  // difference: equal rows leave exactly 0.
  __device__ __forceinline__ double left(int v, float x, float y) const {
    const double w = mp > -INFINITY && x > -INFINITY ? __dmul_rn(weight_table(x, mp, c64, powers), ip) : 0.0;
    if (lq && mq > -INFINITY) return fmax(w - __dmul_rn(weight_table(y, mq, c64, powers), iq), 0.0);
    return v == hot ? 0.0 : w;
  }
  // sum of a segment, in every lane of the warp
  __device__ __forceinline__ double segment(int seg, int V, const uint32_t* bits) const {
    float x[16], y[16];
    load_ids<T>(lp, bits, seg, V, x);
    if (lq) load_ids<T>(lq, nullptr, seg, V, y);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 16; ++j) sum += left(seg * PICK_SEG + lane_id<T>(j), x[j], lq ? y[j] : 0.f);
    return warp_sum(sum);
  }
};

__device__ __forceinline__ double fixed_sum(const double* x, int n, double* sh) {
  double t = 0.0;
  for (int g = threadIdx.x; g < n; g += THREADS) t += x[g];
  return block_sum(t, sh);
}

// The token: each warp adds its segments' weights; the CTA of a request that
// comes last finds the segment in which the sum passes sample_u x total, then
// the id in it.  Bound as norm_kernel is, and by the one CTA at the end: 58 us
// for 48 requests of 248,320 ids with draft rows.
template <typename T>
__global__ void __launch_bounds__(THREADS) pick_kernel(const Params p) {
  __shared__ double sh[WARPS];
  __shared__ int last;
  __shared__ int found_seg, any_seg, found_id, any_id;
  __shared__ double before;
  __shared__ double powers[POWERS];
  fill_powers(powers);
  griddep_wait();
  __syncthreads();
  const int b = blockIdx.y;
  const int n = draft_len(p, b);
  const float z = clean_temperature(p.temperature[b]);
  if (z == 0.f) return;   // greedy: decide_kernel wrote the token
  const Chosen ch = p.chosen[b];
  const int a = ch.row;
  Pick<T> k;
  k.lp = target_row<T>(p, b, a);
  k.lq = nullptr;
  k.mp = ch.mp;
  k.mq = ch.mq;
  k.c64 = 1.44269504088896340736 / (double)z;
  k.powers = powers;
  k.ip = k.iq = 1.0;
  k.hot = -1;
  if (a < n) {
    if (p.draft) {
      k.lq = draft_row<T>(p, b, a);
      const int parts = gridDim.x;   // norm_kernel's grid is this one's
      const double sp = fixed_sum(p.zsum + (size_t)b * parts, parts, sh);
      const double sq = fixed_sum(p.zsum + (size_t)(p.B + b) * parts, parts, sh);
      k.ip = sp > 0.0 ? 1.0 / sp : 0.0;
      k.iq = sq > 0.0 ? 1.0 / sq : 0.0;
    } else {
      k.hot = p.ids[(size_t)b * p.T + a + 1];
    }
  }
  const uint32_t* bits = p.suppress ? p.bits : nullptr;
  double* ws = p.wsum + (size_t)b * p.psegs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = 0; g < p.group; ++g) {
    const int seg = (blockIdx.x * p.group + g) * WARPS + warp;
    if (seg >= p.psegs) break;
    const double sum = k.segment(seg, p.V, bits);
    if (lane == 0) ws[seg] = sum;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&p.ticket[b], 1) == int(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  // The last CTA of the request: total, the segment that the border falls in,
  // then the id inside it.  Which CTA this is changes no sum.
  double total = fixed_sum(ws, p.psegs, sh);
  if (!(total > 0.0)) {
    // nothing left after the draft (equal rows, and a draft that q cannot give):
    // the target's own weights
    k.lq = nullptr;
    k.hot = -1;
    __syncthreads();
    for (int seg = warp; seg < p.psegs; seg += WARPS) {
      const double sum = k.segment(seg, p.V, bits);
      if (lane == 0) ws[seg] = sum;
    }
    __syncthreads();
    total = fixed_sum(ws, p.psegs, sh);
  }
  if (!(total > 0.0)) {
    if (threadIdx.x == 0) p.token[b] = -1;
    return;
  }
  float u = p.sample_u[b];
  u = u > 0.f ? u : 0.f;
  const double border = (double)u * total;
  if (threadIdx.x == 0) {
    found_seg = found_id = 0x7fffffff;
    any_seg = any_id = -1;
  }
  __syncthreads();
  {
    // each thread a run of segments; the first whose sum exceeds the border, or
    // the last that has any, should the sums round below it
    const int per = (p.psegs + THREADS - 1) / THREADS;
    const int g0 = threadIdx.x * per, g1 = min(p.psegs, g0 + per);
    double mine = 0.0;
    for (int g = g0; g < g1; ++g) mine += ws[g];
    const double base = before_me(mine, sh);
    double run = base;
    for (int g = g0; g < g1; ++g) {
      run += ws[g];
      if (!(ws[g] > 0.0)) continue;
      atomicMax(&any_seg, g);
      if (run > border) {
        atomicMin(&found_seg, g);
        break;
      }
    }
    __syncthreads();
    const int chosen = found_seg != 0x7fffffff ? found_seg : any_seg;
    if (chosen >= g0 && chosen < g1) {
      run = base;
      for (int g = g0; g < chosen; ++g) run += ws[g];
      before = border - run;   // what is left of the border inside the segment
    }
    __syncthreads();
    if (threadIdx.x == 0) found_seg = chosen;
    __syncthreads();
  }
  // ids of the segment: each thread two neighbours, the pairs' sums in order
  constexpr int PER = PICK_SEG / THREADS;
  const int w0 = found_seg * PICK_SEG + threadIdx.x * PER;
  double mine = 0.0, piece[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int v = min(w0 + j, p.V - 1);
    float x = to_f<T>(k.lp[v]);
    const float y = k.lq ? to_f<T>(k.lq[v]) : 0.f;
    if (bits && ((bits[v / 32] >> (v & 31)) & 1u)) x = -INFINITY;
    piece[j] = w0 + j < p.V ? k.left(v, x, y) : 0.0;
    mine += piece[j];
  }
  double run = before_me(mine, sh);
  int hit = 0x7fffffff, any = -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    run += piece[j];
    if (piece[j] > 0.0) {
      any = w0 + j;
      if (run > before && hit == 0x7fffffff) hit = w0 + j;
    }
  }
  if (hit != 0x7fffffff) atomicMin(&found_id, hit);
  if (any >= 0) atomicMax(&any_id, any);
  __syncthreads();
  if (threadIdx.x == 0) p.token[b] = found_id != 0x7fffffff ? found_id : any_id;
}

// Segment length of rows_kernel: long enough that a CTA's start-up is small
// beside its loads, short enough that a few rows still fill the card.
inline void geometry(Params* p, int sms) {
  const long long rows = (long long)p->B * p->T + (p->draft ? (long long)p->B * (p->T - 1) : 0);
  int s = MAX_SEG;
  while (s > 4096 && rows * ((p->V + s - 1) / s) < 8ll * sms) s /= 2;
  p->seg = s;
  p->segs = (p->V + s - 1) / s;
  p->psegs = (p->V + PICK_SEG - 1) / PICK_SEG;
  p->words = (p->V + 31) / 32 + 2;
  // likewise for the picked row: more than one segment a warp where there are many
  p->group = 1;
  while (p->group < 8 && (long long)p->B * p->psegs >= 16ll * WARPS * sms * p->group) p->group *= 2;
}

inline size_t round16(size_t x) { return (x + 15) & ~size_t(15); }

inline size_t layout(Params* p, uint8_t* base) {
  const size_t rows = (size_t)p->B * p->T + (p->draft ? (size_t)p->B * (p->T - 1) : 0);
  size_t at = 0;
  auto put = [&](size_t bytes) {
    uint8_t* r = base + at;
    at += round16(bytes);
    return r;
  };
  p->part = reinterpret_cast<float2*>(put(rows * p->segs * sizeof(float2)));
  p->zsum = reinterpret_cast<double*>(put((size_t)2 * p->B * p->psegs * sizeof(double)));
  p->wsum = reinterpret_cast<double*>(put((size_t)p->B * p->psegs * sizeof(double)));
  p->bits = reinterpret_cast<uint32_t*>(put((size_t)p->words * sizeof(uint32_t)));
  p->part_id = reinterpret_cast<int*>(put((size_t)p->B * p->T * p->segs * sizeof(int)));
  p->chosen = reinterpret_cast<Chosen*>(put((size_t)p->B * sizeof(Chosen)));
  p->ticket = reinterpret_cast<int*>(put((size_t)p->B * sizeof(int)));
  return at;
}

template <typename T>
int launch(const Params& p, cudaStream_t stream) {
  const int rows = p.B * p.T + (p.draft ? p.B * (p.T - 1) : 0);
  // The first launch waits for what is before it on the stream as any launch
  // does; the later ones start early and wait for the one before them.
  int st;
  if (p.suppress) {
    mask_kernel<<<(p.words + THREADS - 1) / THREADS, THREADS, 0, stream>>>(p);
    st = host::launch_status();
    if (st != DFL_OK) return st;
    st = host::launch_pdl(rows_kernel<T>, dim3(p.segs, rows), THREADS, 0, stream, p);
  } else {
    rows_kernel<T><<<dim3(p.segs, rows), THREADS, 0, stream>>>(p);
    st = host::launch_status();
  }
  if (st != DFL_OK) return st;
  const int picks = (p.psegs + WARPS * p.group - 1) / (WARPS * p.group);
  st = host::launch_pdl(decide_kernel<T>, dim3(p.B), 32 * DECIDE_WARPS, 0, stream, p);
  if (st != DFL_OK) return st;
  if (p.draft) {   // without the draft's logits there are no sums to take again
    st = host::launch_pdl(norm_kernel<T>, dim3(picks, p.B), THREADS, 0, stream, p);
    if (st != DFL_OK) return st;
  }
  return host::launch_pdl(pick_kernel<T>, dim3(picks, p.B), THREADS, 0, stream, p);
}

// rows <= 65535: the grid's y dimension
inline bool sizes_ok(int B, int T, int V, bool draft) {
  if (B < 0 || T < 1 || T > MAX_BLOCK || V < 1 || V > (1 << 24)) return false;
  return (long long)B * T + (draft ? (long long)B * (T - 1) : 0) <= 65535;
}

}  // namespace smp
}  // namespace dfl

extern "C" size_t dfl_verify_sampled_workspace_bytes(int B, int T, int V, int with_draft, int* status) {
  using namespace dfl;
  int dummy;
  int* st = status ? status : &dummy;
  if (!smp::sizes_ok(B, T, V, with_draft != 0)) {
    *st = DFL_ERR_BAD_SHAPE;
    return 0;
  }
  int dev, sms;
  *st = host::current_device(&dev, &sms);
  if (*st != DFL_OK) return 0;
  smp::Params p;
  p.B = B;
  p.T = T;
  p.V = V;
  p.draft = with_draft ? &p : nullptr;
  smp::geometry(&p, sms);
  return smp::layout(&p, nullptr);
}

extern "C" int dfl_verify_accept_sampled(const void* logits, const void* draft_logits, int dtype,
                                         const int32_t* verify_ids, const float* accept_u,
                                         const float* sample_u, const float* temperature,
                                         const int32_t* draft_lens, const uint8_t* suppress, int32_t* acceptance,
                                         int32_t* next_token, float* draft_prob, size_t ld_logits, size_t bs_logits,
                                         size_t ld_draft, size_t bs_draft, int B, int T, int V,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dfl;
  if (!smp::sizes_ok(B, T, V, draft_logits != nullptr)) return DFL_ERR_BAD_SHAPE;
  if (dtype < 0 || dtype > 2) return DFL_ERR_UNSUPPORTED;
  const size_t far = (size_t)1 << 40;
  if (ld_logits > far || bs_logits > far || ld_draft > far || bs_draft > far) return DFL_ERR_BAD_SHAPE;
  if (B == 0) return DFL_OK;
  if (!logits || !sample_u || !temperature || !acceptance || !next_token) return DFL_ERR_NULL_POINTER;
  if (T > 1 && (!verify_ids || !accept_u || !draft_prob)) return DFL_ERR_NULL_POINTER;
  const uintptr_t esz = dtype == 2 ? 4 : 2;
  if (!host::aligned(logits, esz) || !host::aligned(draft_logits, esz)) return DFL_ERR_MISALIGNED;
  int dev, sms;
  const int st = host::current_device(&dev, &sms);
  if (st != DFL_OK) return st;
  smp::Params p;
  p.logits = logits;
  p.draft = draft_logits;
  p.ids = verify_ids;
  p.accept_u = accept_u;
  p.sample_u = sample_u;
  p.temperature = temperature;
  p.lens = draft_lens;
  p.suppress = suppress;
  p.accepted = acceptance;
  p.token = next_token;
  p.draft_prob = draft_prob;
  p.ld = (long long)ld_logits;
  p.ldd = (long long)ld_draft;
  p.bs = (long long)bs_logits;
  p.bsd = (long long)bs_draft;
  p.B = B;
  p.T = T;
  p.V = V;
  smp::geometry(&p, sms);
  if (!workspace || !host::aligned(workspace, 16)) return workspace ? DFL_ERR_MISALIGNED : DFL_ERR_WORKSPACE;
  if (workspace_bytes < smp::layout(&p, reinterpret_cast<uint8_t*>(workspace))) return DFL_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return smp::launch<__nv_bfloat16>(p, s);
    case 1: return smp::launch<__half>(p, s);
    default: return smp::launch<float>(p, s);
  }
}
