// Routing of tokens to experts (sm_100a): for each token's logits l [E]
//     s = sigmoid(l) or softmax(l);  c = s + bias            (the bias only chooses)
//     groups of E / n_groups experts: score = sum of the group's two largest c,
//     or its largest; the topk_groups best groups stay
//     ids = top_k experts of those by c (largest first, ties to the lower id)
//     w = s[ids] (/ sum of them), x scale
// An expert whose logit is NaN or -inf cannot be had: its weight is 0 and it
// only fills a slot that no other expert of the kept groups is left for, so
// ids are always distinct and in [0, E).
//
// Scores are 64 bits: which experts are kept turns on small differences of s +
// bias, and the weights come out of the same numbers.
//
// The router of mlx-lm's MoE blocks (third party), reached with SwitchGLU from
// dflash_mlx/engine/target_qwen_gdn.py:863-865.

namespace dfl {
namespace rt {

constexpr int MAX_TOP_K = 32;      // one lane per kept expert
constexpr int MAX_EXPERTS = 4096;

struct Params {
  const void* logits;  // [T, E], rows of ld
  const float* bias;   // [E] or null
  float* weights;      // [T, k]
  int32_t* ids;        // [T, k]
  long long ld;
  int T, E, k, groups, topk_groups;
  int sigmoid, top2, renorm;
  float scale;
};

// (value desc, id asc); the sentinel (-inf, INT_MAX) loses against every expert
__device__ __forceinline__ bool ahead(double v, int e, double w, int f) { return v > w || (v == w && e < f); }

__device__ __forceinline__ void warp_best(double* v, int* e) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(0xffffffffu, *v, o);
    const int oe = __shfl_xor_sync(0xffffffffu, *e, o);
    if (ahead(ov, oe, *v, *e)) {
      *v = ov;
      *e = oe;
    }
  }
}

// One warp per token; its scores and choices stand in shared memory.
template <typename T>
__global__ void route_kernel(const Params p) {
  extern __shared__ double sh_rt[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * (blockDim.x >> 5) + warp;
  if (t >= p.T) return;
  double* s = sh_rt + (size_t)warp * (2 * p.E + p.groups);  // scores
  double* c = s + p.E;                                      // choices; -inf: cannot be had
  double* gs = c + p.E;                                     // group scores
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)t * p.ld;
  float mx = -INFINITY;
  if (!p.sigmoid) {
    for (int e = lane; e < p.E; e += 32) mx = fmaxf(mx, smp::to_f<T>(row[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  double sum = 0.0;
  for (int e = lane; e < p.E; e += 32) {
    const float x = smp::to_f<T>(row[e]);
    const bool have = x > -INFINITY;   // false for NaN
    double w = 0.0;
    if (have) w = p.sigmoid ? 1.0 / (1.0 + exp(-(double)x)) : smp::weight(x, mx, 1.0);
    s[e] = w;
    c[e] = have ? 0.0 : -INFINITY;
    sum += w;
  }
  double inv = 1.0;
  if (!p.sigmoid) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    inv = sum > 0.0 ? 1.0 / sum : 0.0;
  }
  for (int e = lane; e < p.E; e += 32) {
    const double w = p.sigmoid ? s[e] : s[e] * inv;
    s[e] = w;
    double x = w + (p.bias ? (double)p.bias[e] : 0.0);
    if (c[e] != 0.0 || !(x == x)) x = -INFINITY;
    c[e] = x;
  }
  __syncwarp();
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    for (int g = 0; g < p.groups; ++g) {
      double b0 = -INFINITY, b1 = -INFINITY;
      for (int e = lane; e < size; e += 32) {
        const double x = c[g * size + e];
        if (x > b0) {
          b1 = b0;
          b0 = x;
        } else if (x > b1) {
          b1 = x;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double o0 = __shfl_xor_sync(0xffffffffu, b0, o);
        const double o1 = __shfl_xor_sync(0xffffffffu, b1, o);
        b1 = fmax(fmin(b0, o0), fmax(b1, o1));
        b0 = fmax(b0, o0);
      }
      if (lane == 0) gs[g] = p.top2 && b1 > -INFINITY ? b0 + b1 : b0;
    }
    __syncwarp();
    // the best groups, one after the other; what is not among them is closed
    // (lowered to a value that is told from "cannot be had" by its id order alone)
    for (int j = 0; j < p.topk_groups; ++j) {
      double b = -INFINITY;
      int bg = 0x7fffffff;
      for (int g = lane; g < p.groups; g += 32)
        if (gs[g] == gs[g] && ahead(gs[g], g, b, bg)) {
          b = gs[g];
          bg = g;
        }
      warp_best(&b, &bg);
      if (lane == 0) gs[bg] = NAN;   // taken
      __syncwarp();
    }
    for (int e = lane; e < p.E; e += 32)
      if (gs[e / size] == gs[e / size]) c[e] = NAN;   // a group that was not taken
    __syncwarp();
  }
  double mine = 0.0;
  int my_id = 0;
  double total = 0.0;
  for (int j = 0; j < p.k; ++j) {
    double b = -INFINITY;
    int be = 0x7fffffff;
    for (int e = lane; e < p.E; e += 32)
      if (c[e] == c[e] && ahead(c[e], e, b, be)) {
        b = c[e];
        be = e;
      }
    warp_best(&b, &be);
    if (lane == 0) c[be] = NAN;   // taken
    const double w = b > -INFINITY ? s[be] : 0.0;
    total += w;
    if (lane == j) {
      mine = w;
      my_id = be;
    }
    __syncwarp();
  }
  if (lane < p.k) {
    if (p.renorm) mine = total > 0.0 ? mine / total : 0.0;
    p.weights[(size_t)t * p.k + lane] = float(mine * (double)p.scale);
    p.ids[(size_t)t * p.k + lane] = my_id;
  }
}

// The same in registers, a warp per token, for up to 32 EPL experts: lane l holds
// experts l EPL .. l EPL + EPL - 1, so that ids rise with the lanes and a group
// of neighbours is a run of lanes.  Every group's two best are found at once
// (log2 of its lanes shuffles) and a group's rank is the number of groups
// ahead of it.  Experts are picked by an order-preserving 64-bit image of c: the
// largest high word, then the largest low word under it (two reductions over
// the warp), the first lane that has both, its first expert.  Groups have to
// be runs of whole lanes: n_groups a power of two up to 32 and E = 32 EPL, or
// one group.
//
// Bound by the instructions of the 64-bit scores and of the k rounds (8191 tokens
// of 256 experts: 27 us, where their 4.7 MB would take 0.7).
template <typename T, int EPL>
__global__ void __launch_bounds__(128) route_lanes_kernel(const Params p) {
  constexpr unsigned ALL = 0xffffffffu;
  constexpr unsigned long long GONE = 0;   // below the image of -inf
  constexpr unsigned long long NONE = ~0xfff0000000000000ull;   // the image of -inf: cannot be had
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)t * p.ld;
  float x[EPL];
  float bias[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    x[i] = e < p.E ? smp::to_f<T>(row[e]) : -INFINITY;
    bias[i] = p.bias && e < p.E ? p.bias[e] : 0.f;
  }
  double s[EPL];
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) s[i] = x[i] > -INFINITY ? __drcp_rn(1.0 + exp(-(double)x[i])) : 0.0;
  } else {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, x[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, o));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      s[i] = smp::weight(x[i], mx, 1.0);
      if (!(x[i] > -INFINITY)) s[i] = 0.0;
      sum += s[i];
    }
    sum = smp::warp_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) s[i] *= inv;
  }
  unsigned long long key[EPL];
  double b0 = -INFINITY, b1 = -INFINITY;   // this lane's two largest c
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    double c = s[i] + (double)bias[i];
    if (!(x[i] > -INFINITY) || !(c == c)) c = -INFINITY;
    c += 0.0;                              // -0 and +0 tie
    const long long bits = __double_as_longlong(c);
    key[i] = (unsigned long long)(bits ^ ((bits >> 63) | (long long)0x8000000000000000ull));
    if (lane * EPL + i >= p.E) key[i] = GONE;
    b1 = fmax(b1, fmin(b0, c));
    b0 = fmax(b0, c);
  }
  if (p.groups > 1) {
    const int lanes = 32 / p.groups;
    for (int o = 1; o < lanes; o *= 2) {
      const double o0 = __shfl_xor_sync(ALL, b0, o), o1 = __shfl_xor_sync(ALL, b1, o);
      b1 = fmax(fmin(b0, o0), fmax(b1, o1));
      b0 = fmax(b0, o0);
    }
    const double mine = p.top2 && b1 > -INFINITY ? b0 + b1 : b0;
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double other = __shfl_sync(ALL, mine, g * lanes);
      rank += other > mine || (other == mine && g < lane / lanes);
    }
    if (rank >= p.topk_groups) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) key[i] = GONE;
    }
  }
  double w = 0.0, total = 0.0;
  int id = 0;
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = key[0];
    double bs = s[0];
    int bi = 0;
#pragma unroll
    for (int i = 1; i < EPL; ++i)
      if (key[i] > best) {
        best = key[i];
        bs = s[i];
        bi = i;
      }
    const unsigned hi = unsigned(best >> 32), top = __reduce_max_sync(ALL, hi);
    const unsigned lo = hi == top ? unsigned(best) : 0u, low = __reduce_max_sync(ALL, lo);
    const int from = __ffs(__ballot_sync(ALL, hi == top && unsigned(best) == low)) - 1;
    double ws = __shfl_sync(ALL, best > NONE ? bs : 0.0, from);
    const int e = __shfl_sync(ALL, lane * EPL + bi, from);
    if (lane == from) {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i == bi) key[i] = GONE;
    }
    total += ws;
    if (lane == j) {
      w = ws;
      id = e;
    }
  }
  if (lane < p.k) {
    if (p.renorm) w = total > 0.0 ? w / total : 0.0;
    p.weights[(size_t)t * p.k + lane] = float(w * (double)p.scale);
    p.ids[(size_t)t * p.k + lane] = id;
  }
}

// The register form where the sizes fit it, else the one on shared memory.
// Measured at 256 experts, 8 groups, top 8: 16 tokens 6.2 us for 14.4 us, 8191
// tokens 27 us for 45 us.
template <typename T>
bool launch_lanes(const Params& p, cudaStream_t stream) {
  const bool runs = (p.groups & (p.groups - 1)) == 0 && p.groups <= 32;
  const int grid = (p.T + 3) / 4;
  if (p.groups == 1 ? p.E <= 64 : runs && p.E == 64) {
    route_lanes_kernel<T, 2><<<grid, 128, 0, stream>>>(p);
  } else if (p.groups == 1 ? p.E <= 128 : runs && p.E == 128) {
    route_lanes_kernel<T, 4><<<grid, 128, 0, stream>>>(p);
  } else if (p.groups == 1 ? p.E <= 256 : runs && p.E == 256) {
    route_lanes_kernel<T, 8><<<grid, 128, 0, stream>>>(p);
  } else if (p.groups == 1 ? p.E <= 512 : runs && p.E == 512) {
    route_lanes_kernel<T, 16><<<grid, 128, 0, stream>>>(p);
  } else {
    return false;
  }
  return true;
}

template <typename T>
int launch(const Params& p, int dev, cudaStream_t stream) {
  if (launch_lanes<T>(p, stream)) return host::launch_status();
  static std::atomic<uint64_t> done{0};
  const size_t per = (size_t)(2 * p.E + p.groups) * sizeof(double);
  int warps = int((size_t)48 * 1024 / per);
  warps = warps < 1 ? 1 : (warps > 8 ? 8 : warps);
  const int st = host::ensure_smem(route_kernel<T>, 3 * MAX_EXPERTS * int(sizeof(double)), dev, done);
  if (st != DFL_OK) return st;
  route_kernel<T><<<(p.T + warps - 1) / warps, 32 * warps, per * warps, stream>>>(p);
  return host::launch_status();
}

}  // namespace rt
}  // namespace dfl

extern "C" int dfl_moe_route_experts(const void* logits, int dtype, size_t ld, const float* bias, int T, int E,
                                     int top_k, int n_groups, int topk_groups, int flags, float scale,
                                     float* weights, int32_t* topk_ids, void* stream) {
  using namespace dfl;
  if (T < 0 || E < 1 || E > rt::MAX_EXPERTS || top_k < 1 || top_k > rt::MAX_TOP_K) return DFL_ERR_BAD_SHAPE;
  if (n_groups < 1 || n_groups > E || E % n_groups != 0 || topk_groups < 1 || topk_groups > n_groups)
    return DFL_ERR_BAD_SHAPE;
  if (top_k > topk_groups * (E / n_groups) || ld < (size_t)E || ld > (size_t)1 << 40) return DFL_ERR_BAD_SHAPE;
  if (dtype < 0 || dtype > 2 || (flags & ~(DFL_ROUTE_SIGMOID | DFL_ROUTE_GROUP_TOP2 | DFL_ROUTE_RENORM)))
    return DFL_ERR_UNSUPPORTED;
  if (T == 0) return DFL_OK;
  if (!logits || !weights || !topk_ids) return DFL_ERR_NULL_POINTER;
  if (!host::aligned(logits, dtype == 2 ? 4 : 2)) return DFL_ERR_MISALIGNED;
  int dev, sms;
  const int st = host::current_device(&dev, &sms);
  if (st != DFL_OK) return st;
  rt::Params p;
  p.logits = logits;
  p.bias = bias;
  p.weights = weights;
  p.ids = topk_ids;
  p.ld = (long long)ld;
  p.T = T;
  p.E = E;
  p.k = top_k;
  p.groups = n_groups;
  p.topk_groups = topk_groups;
  p.sigmoid = (flags & DFL_ROUTE_SIGMOID) != 0;
  p.top2 = (flags & DFL_ROUTE_GROUP_TOP2) != 0;
  p.renorm = (flags & DFL_ROUTE_RENORM) != 0;
  p.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return rt::launch<__nv_bfloat16>(p, dev, s);
    case 1: return rt::launch<__half>(p, dev, s);
    default: return rt::launch<float>(p, dev, s);
  }
}

namespace dfl {
namespace rt {

// The route table of moe::route_kernel (same layout and order) from given ids;
// a pair whose id is outside [0, E) sets the device error word and is left out.
__global__ void table_kernel(const int32_t* ids_in, int T, int E, int k, int32_t* table) {
  extern __shared__ int sh_tb[];
  int* cnt = sh_tb;              // [E]
  int* start = cnt + E;          // [E]
  int* ids = start + E;          // [T * k]
  const int tid = threadIdx.x, pairs = T * k;
  for (int e = tid; e < E; e += blockDim.x) cnt[e] = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += blockDim.x) {
    int e = ids_in[i];
    if (e < 0 || e >= E) {
      atomicExch(&g_device_error, kDevBadInput);
      e = -1;
    } else {
      atomicAdd(&cnt[e], 1);
    }
    ids[i] = e;
  }
  __syncthreads();
  if (tid < 32) {
    // problem numbers of the active experts, in increasing id order
    int base = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + tid;
      const bool on = e < E && cnt[e] > 0;
      const unsigned m = __ballot_sync(0xffffffffu, on);
      if (e < E) start[e] = on ? base + __popc(m & ((1u << tid) - 1u)) : -1;
      base += __popc(m);
    }
    if (tid == 0) table[0] = base;
  }
  __syncthreads();
  for (int e = tid; e < E; e += blockDim.x) {
    const int pi = start[e];
    if (pi >= 0) {
      table[1 + pi] = e;
      table[1 + E + pi] = min(cnt[e], moe::MAX_TOKENS);
    }
  }
  for (int pr = tid; pr < pairs; pr += blockDim.x) {
    const int e = ids[pr];
    if (e < 0) continue;
    int m = 0;
    for (int q = 0; q < pr; ++q) m += (ids[q] == e);
    if (m >= moe::MAX_TOKENS) {   // the same expert twice for one token
      atomicExch(&g_device_error, kDevBadInput);
      continue;
    }
    const int pi = start[e];
    table[1 + 2 * E + pi * 16 + m] = pr / k;          // token row
    table[1 + 2 * E + 16 * E + pi * 16 + m] = pr;     // pair row
  }
}

}  // namespace rt
}  // namespace dfl

extern "C" int dfl_moe_route_table(const int32_t* topk_ids, int T, int top_k, int E, int32_t* route_table,
                                   void* stream) {
  using namespace dfl;
  if (T < 1 || T > moe::MAX_TOKENS || E < 1 || E > rt::MAX_EXPERTS || top_k < 1 || top_k > moe::MAX_K)
    return DFL_ERR_BAD_SHAPE;
  if (!topk_ids || !route_table) return DFL_ERR_NULL_POINTER;
  int dev, sms;
  const int st = host::current_device(&dev, &sms);
  if (st != DFL_OK) return st;
  const size_t smem = (size_t)(2 * E + T * top_k) * sizeof(int);   // 34 KB at most
  rt::table_kernel<<<1, 256, smem, reinterpret_cast<cudaStream_t>(stream)>>>(topk_ids, T, E, top_k, route_table);
  return host::launch_status();
}
