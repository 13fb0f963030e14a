// Verification of drafted tokens against the target's distribution, from given
// uniforms (speculative sampling), with the behaviour log-probs of the tokens it
// leaves.
//
// Per sequence: target rows x_0..x_K, draft rows y_0..y_{K-1}, drafts d_0..d_{K-1}
// (a negative one ends the draft at length L), uniforms u_0..u_K.
//   p_j = softmax(x_j / T), q_j = softmax(y_j / T) (or one-hot at d_j)
//   d_j is accepted while u_j q_j(d_j) < p_j(d_j);  n = the first that is not, or L
//   rest = max(p_n - q_n, 0) after a rejection (p_n where that has no mass), p_L else
//   the last token: the first v whose running sum of rest exceeds u_K sum(rest)
// Greedy: d_j is accepted while it is x_j's first maximum; the last token is x_n's.
//
// A token is decided by where a running sum over the vocabulary passes a border,
// and there are as many borders as entries: float32 sums (1e-7 of the whole) would
// pass a wrong one every some ten rows of 150,000 entries.  Exponentials and sums
// are therefore float64, the exponential a polynomial good to 1.1e-12.
//
// Rows are cut into chunks, so that a single sequence fills the chip:
//   1. verify_stats: every needed row's chunks: maximum, sum of exponentials
//   2. verify_decide: a workgroup per sequence joins them and finds n
//   3. verify_rest: after a rejection, the mass of rest in every chunk of row n
//   4. verify_draw: a workgroup per sequence finds the chunk, then the entry
#include "slab_common.hpp"

namespace rrl {
namespace {

constexpr int kVT = 256;        // threads of a workgroup
constexpr int kChunk = 4096;    // entries of a chunk

// 2^r for |r| <= 1/2: the polynomial through 2^r at the nine Chebyshev nodes of
// that interval, within 1.1e-12 of it, relative.
__device__ __forceinline__ double exp2_poly(double r) {
  double p = 0x1.63d1363942fefp-20;
  p = fma(p, r, 0x1.00dc4a534288bp-16);
  p = fma(p, r, 0x1.4308ac85a7a46p-13);
  p = fma(p, r, 0x1.5d8745a7281dep-10);
  p = fma(p, r, 0x1.3b2ab7181b773p-7);
  p = fma(p, r, 0x1.c6b08dd6fd237p-5);
  p = fma(p, r, 0x1.ebfbdff823cedp-3);
  p = fma(p, r, 0x1.62e42fef84cf0p-1);
  return fma(p, r, 1.0);
}

// 2^t for t <= 0 (0 for -inf).  Below -1000 the result, under 1e-301 beside a
// maximum of 1, is taken as 2^-1000.. of the clamped t: it is left at 0.
__device__ __forceinline__ double exp2_neg(double t) {
  if (!(t > -1000.0)) return 0.0;
  const double n = rint(t);
  return ldexp(exp2_poly(t - n), (int)n);
}

struct VerifyArgs {
  const char *x, *y;            // target, draft logits (y may be null)
  int64_t xs_b, xs_k, ys_b, ys_k;  // strides (elements)
  const void* drafts;
  int drafts_dt;
  int64_t ds_b, ds_k;
  const float* u;               // [B, K + 1]
  int64_t B, K, V;
  double c;                     // log2(e) / T
  int greedy;
  int rows;                     // rows per sequence: K + 1 target rows, then the draft's
  int chunks;
  int64_t* token_out;           // [B, K + 1]
  int64_t* count_out;           // [B]
  float* logp_out;              // [B, K + 1]
};

struct ChunkStat {
  double s;    // sum of 2^(c (x - m))
  float m;     // maximum; +inf: the chunk holds NaN or +inf
  int32_t at;  // first index of the maximum
};
struct RowStat {
  double s;
  float m;  // +inf: a row that has no distribution
  int32_t at;
};
enum : int32_t { REST_P = 0, REST_PQ = 1, REST_P_WITHOUT_DRAFT = 2, REST_BAD = 3 };
struct Plan {
  int32_t n, rest;
};

struct Ws {
  ChunkStat* stat;  // [B, rows, chunks]
  RowStat* row;     // [B, rows]
  double* mass;     // [B, chunks]
  Plan* plan;       // [B]
};

template <class Tag>
__device__ __forceinline__ const char* target_row(const VerifyArgs& a, int64_t b, int64_t j) {
  return a.x + (b * a.xs_b + j * a.xs_k) * (16 / Pack16<Tag>::EPV);
}
template <class Tag>
__device__ __forceinline__ const char* draft_row(const VerifyArgs& a, int64_t b, int64_t j) {
  return a.y + (b * a.ys_b + j * a.ys_k) * (16 / Pack16<Tag>::EPV);
}
__device__ __forceinline__ int64_t draft_at(const VerifyArgs& a, int64_t b, int64_t j) {
  return load_index(a.drafts, a.drafts_dt, b * a.ds_b + j * a.ds_k);
}

// A row may start at any element: these 16 bytes are one global_load_dwordx4 at
// any address.
struct __attribute__((packed, aligned(2))) Any16 {
  u32x4 v;
};

// Entries i..i+EPV of a row, -inf past its end.
template <class Tag>
__device__ __forceinline__ void load_entries(const char* row, int64_t i, int64_t V,
                                             float (&x)[Pack16<Tag>::EPV]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (i + EPV <= V) {
    Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ)->v, x);
    return;
  }
#pragma unroll
  for (int k = 0; k < EPV; ++k) {
    x[k] = -M<float>::inf();
    if (i + k < V) {
      if constexpr (SZ == 4) {
        x[k] = reinterpret_cast<const float*>(row)[i + k];
      } else {
        x[k] = Pack16<Tag>::one(reinterpret_cast<const uint16_t*>(row)[i + k]);
      }
    }
  }
}
template <class Tag>
__device__ __forceinline__ float load_entry(const char* row, int64_t i) {
  if constexpr (16 / Pack16<Tag>::EPV == 4) return reinterpret_cast<const float*>(row)[i];
  else return Pack16<Tag>::one(reinterpret_cast<const uint16_t*>(row)[i]);
}

// ---- 1: chunks -----------------------------------------------------------------------

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_stats_kernel(VerifyArgs a, Ws ws) {
  constexpr int EPV = Pack16<Tag>::EPV, NS = kChunk / (kVT * EPV);
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const int64_t id = blockIdx.x;
  const int chunk = (int)(id % a.chunks);
  const int64_t rid = id / a.chunks, b = rid / a.rows;
  const int r = (int)(rid % a.rows);
  // target row j serves only if the j drafts before it exist, draft row j also its own
  const bool is_draft = r > a.K;
  const int j = is_draft ? r - (int)a.K - 1 : r;
  for (int k = 0; k < j + (is_draft ? 1 : 0); ++k)
    if (draft_at(a, b, k) < 0) return;
  const char* row = is_draft ? draft_row<Tag>(a, b, j) : target_row<Tag>(a, b, j);

  float x[NS][EPV];
  const int64_t lo = (int64_t)chunk * kChunk + t * EPV;
#pragma unroll
  for (int s = 0; s < NS; ++s) load_entries<Tag>(row, lo + s * kVT * EPV, a.V, x[s]);
  float m = -M<float>::inf();
  bool bad = false;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int k = 0; k < EPV; ++k) {
      m = fmaxf(m, x[s][k]);
      bad |= !(x[s][k] < M<float>::inf());  // NaN or +inf
    }
  if (bad) m = M<float>::inf();
  __shared__ float sm[kVT / 64];
  __shared__ double ss[kVT / 64];
  __shared__ int sat[kVT / 64];
  m = wave_max_dpp(m);
  if (lane == 0) sm[wv] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  int at = 0x7fffffff;
  double sum = 0.0;
  if (m > -M<float>::inf() && m < M<float>::inf()) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int k = 0; k < EPV; ++k) sum += exp2_neg(((double)x[s][k] - (double)m) * a.c);
    if (a.greedy) {
#pragma unroll
      for (int s = NS - 1; s >= 0; --s)
#pragma unroll
        for (int k = EPV - 1; k >= 0; --k)
          if (x[s][k] == m) at = (int)(lo + s * kVT * EPV + k);
    }
  }
  sum = wave_sum(sum);
  at = wave_min_dpp(at);
  if (lane == 0) {
    ss[wv] = sum;
    sat[wv] = at;
  }
  __syncthreads();
  if (t == 0)
    ws.stat[id] = ChunkStat{(ss[0] + ss[1]) + (ss[2] + ss[3]), m,
                            min(min(sat[0], sat[1]), min(sat[2], sat[3]))};
}

// ---- 2: rows, and how far the draft is accepted -----------------------------------------

// Joins the chunks of one row; the whole wave takes part.
__device__ __forceinline__ RowStat join_row(const ChunkStat* st, int chunks, double c) {
  const int lane = threadIdx.x & 63;
  float m = -M<float>::inf();
  for (int k = lane; k < chunks; k += 64) m = fmaxf(m, st[k].m);
  m = wave_max_dpp(m);
  double s = 0.0;
  int at = 0x7fffffff;
  if (m == -M<float>::inf()) m = M<float>::inf();  // nothing is possible: no distribution
  if (m < M<float>::inf())
    for (int k = lane; k < chunks; k += 64) {
      s += st[k].s * exp2_neg(((double)st[k].m - (double)m) * c);
      if (st[k].m == m) at = min(at, st[k].at);
    }
  return RowStat{wave_sum(s), m, wave_min_dpp(at)};
}

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_decide_kernel(VerifyArgs a, Ws ws) {
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  __shared__ int sh_len, sh_n, sh_rest;
  if (t == 0) {
    int len = 0;
    while (len < a.K && draft_at(a, b, len) >= 0) ++len;
    sh_len = len;
    sh_n = len;
    sh_rest = REST_P;
  }
  __syncthreads();
  const int L = sh_len;
  const bool has_q = a.y != nullptr;
  RowStat* row = ws.row + b * a.rows;
  for (int r = wv; r < a.rows; r += kVT / 64) {
    const bool is_draft = r > a.K;
    if (is_draft ? r - (int)a.K - 1 >= L : r > L) continue;
    const RowStat s = join_row(ws.stat + (b * a.rows + r) * a.chunks, a.chunks, a.c);
    if (lane == 0) row[r] = s;
  }
  __syncthreads();
  // positions in turn, kVT at a time: the first that does not accept its draft
  for (int j0 = 0; j0 < L && sh_n == L; j0 += kVT) {
    const int j = j0 + t;
    int rest = -1;
    if (j < L) {
      const RowStat p = row[j];
      const int64_t d = draft_at(a, b, j);
      if (!(p.m < M<float>::inf()) || d >= a.V) {
        rest = REST_BAD;
      } else if (a.greedy) {
        if (d != p.at) rest = REST_P;
      } else {
        const double px =
            exp2_neg(((double)load_entry<Tag>(target_row<Tag>(a, b, j), d) - (double)p.m) * a.c) / p.s;
        double qx = 1.0;
        bool bad = false;
        if (has_q) {
          const RowStat q = row[a.K + 1 + j];
          bad = !(q.m < M<float>::inf());
          if (!bad)
            qx = exp2_neg(((double)load_entry<Tag>(draft_row<Tag>(a, b, j), d) - (double)q.m) * a.c) /
                 q.s;
        }
        if (bad) rest = REST_BAD;
        else if (!((double)a.u[b * (a.K + 1) + j] * qx < px))
          rest = has_q ? REST_PQ : REST_P_WITHOUT_DRAFT;
      }
    }
    __syncthreads();
    if (rest >= 0) atomicMin(&sh_n, j);
    __syncthreads();
    if (rest >= 0 && sh_n == j) sh_rest = rest;
    __syncthreads();
  }
  if (t == 0) {
    if (sh_n == L && !(row[L].m < M<float>::inf())) sh_rest = REST_BAD;
    ws.plan[b] = Plan{sh_n, sh_rest};
  }
}

// ---- 3 and 4: the last token -------------------------------------------------------------

// What an entry of the deciding row weighs.
template <class Tag>
struct Rest {
  const char *x, *y;
  double mp, mq, ip, iq, c;  // maxima and 1 / sums
  int64_t skip;              // an entry without mass (the rejected draft), or -1
  __device__ __forceinline__ void weights(int64_t i, int64_t V, double (&w)[Pack16<Tag>::EPV]) const {
    constexpr int EPV = Pack16<Tag>::EPV;
    float v[EPV];
    load_entries<Tag>(x, i, V, v);
#pragma unroll
    for (int k = 0; k < EPV; ++k) w[k] = exp2_neg(((double)v[k] - mp) * c) * ip;
    if (y) {
      load_entries<Tag>(y, i, V, v);
#pragma unroll
      for (int k = 0; k < EPV; ++k)
        w[k] = fmax(w[k] - exp2_neg(((double)v[k] - mq) * c) * iq, 0.0);
    }
#pragma unroll
    for (int k = 0; k < EPV; ++k)
      if (i + k == skip) w[k] = 0.0;
  }
};

template <class Tag>
__device__ __forceinline__ Rest<Tag> rest_of(const VerifyArgs& a, const Ws& ws, int64_t b, int n,
                                             int kind) {
  const RowStat p = ws.row[b * a.rows + n];
  Rest<Tag> r{target_row<Tag>(a, b, n), nullptr, p.m, 0.0, 1.0 / p.s, 0.0, a.c, -1};
  if (kind == REST_PQ) {
    const RowStat q = ws.row[b * a.rows + a.K + 1 + n];
    r.y = draft_row<Tag>(a, b, n);
    r.mq = q.m;
    r.iq = 1.0 / q.s;
  } else if (kind == REST_P_WITHOUT_DRAFT) {
    r.skip = draft_at(a, b, n);
  }
  return r;
}

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_rest_kernel(VerifyArgs a, Ws ws) {
  constexpr int EPV = Pack16<Tag>::EPV, NS = kChunk / (kVT * EPV);
  const int64_t b = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks), t = threadIdx.x;
  const Plan pl = ws.plan[b];
  if (pl.rest != REST_PQ && pl.rest != REST_P_WITHOUT_DRAFT) return;
  const Rest<Tag> r = rest_of<Tag>(a, ws, b, pl.n, pl.rest);
  double sum = 0.0;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    double w[EPV];
    r.weights((int64_t)chunk * kChunk + (s * kVT + t) * EPV, a.V, w);
#pragma unroll
    for (int k = 0; k < EPV; ++k) sum += w[k];
  }
  __shared__ double ss[kVT / 64];
  sum = wave_sum(sum);
  if ((t & 63) == 0) ss[t >> 6] = sum;
  __syncthreads();
  if (t == 0) ws.mass[blockIdx.x] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// Inclusive running sum over the workgroup; total to every thread.
__device__ __forceinline__ double block_scan(double v, double& total, double* sh) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63) sh[wv] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int k = 0; k < kVT / 64; ++k) {
    if (k < wv) before += sh[k];
    total += sh[k];
  }
  return before + v;
}

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_draw_kernel(VerifyArgs a, Ws ws) {
  constexpr int EPV = Pack16<Tag>::EPV, NS = kChunk / (kVT * EPV);
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  const Plan pl = ws.plan[b];
  const int n = pl.n;
  const RowStat* rows = ws.row + b * a.rows;
  __shared__ double sh[kVT / 64];
  __shared__ int first, last;  // chunk, then entry within the chunk
  __shared__ double sh_rem;
  int64_t token = -1;
  if (pl.rest != REST_BAD && a.greedy) {
    token = rows[n].at;
  } else if (pl.rest != REST_BAD) {
    const double u = a.u[b * (a.K + 1) + a.K];
    int kind = pl.rest;
    double total = 0.0;
    if (kind != REST_P) {
      double v = 0.0;
      for (int k = t; k < a.chunks; k += kVT) v += ws.mass[b * a.chunks + k];
      block_scan(v, total, sh);
      if (!(total > 0.0)) kind = REST_P;  // the two rows are equal to within rounding
    }
    const Rest<Tag> r = rest_of<Tag>(a, ws, b, n, kind);
    const ChunkStat* st = ws.stat + (b * a.rows + n) * a.chunks;
    auto chunk_mass = [&](int k) {
      if (k >= a.chunks) return 0.0;
      if (kind != REST_P) return ws.mass[b * a.chunks + k];
      return st[k].s * exp2_neg(((double)st[k].m - r.mp) * a.c) * r.ip;
    };
    if (kind == REST_P) {
      double v = 0.0;
      for (int k = t; k < a.chunks; k += kVT) v += chunk_mass(k);
      block_scan(v, total, sh);
    }
    const double border = u * total;
    // the first chunk whose running sum passes the border, else the last with any mass
    if (t == 0) {
      first = 0x7fffffff;
      last = -1;
    }
    double before = 0.0;
    __syncthreads();
    for (int k0 = 0; k0 < a.chunks; k0 += kVT) {
      const double w = chunk_mass(k0 + t);
      double sum;
      const double incl = block_scan(w, sum, sh) + before;
      if (w > 0.0) {
        atomicMax(&last, k0 + t);
        if (incl > border) atomicMin(&first, k0 + t);
      }
      __syncthreads();
      if (first == k0 + t) sh_rem = border - (incl - w);
      before += sum;
      __syncthreads();
      if (first != 0x7fffffff) break;
    }
    const bool over = first == 0x7fffffff;
    const int chunk = over ? last : first;
    const double rem = over ? M<double>::inf() : sh_rem;
    __syncthreads();
    if (t == 0) {
      first = 0x7fffffff;
      last = -1;
    }
    before = 0.0;
    __syncthreads();
#pragma unroll 1
    for (int s = 0; s < NS; ++s) {
      double w[EPV], mine = 0.0, sum;
      const int e0 = (s * kVT + t) * EPV;
      r.weights((int64_t)chunk * kChunk + e0, a.V, w);
#pragma unroll
      for (int k = 0; k < EPV; ++k) mine += w[k];
      double at = block_scan(mine, sum, sh) - mine + before;
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        at += w[k];
        if (w[k] > 0.0) {
          atomicMax(&last, e0 + k);
          if (at > rem) atomicMin(&first, e0 + k);
        }
      }
      before += sum;
    }
    __syncthreads();
    token = (int64_t)chunk * kChunk + (first != 0x7fffffff ? first : last);
  }
  // the accepted drafts, the last token, and nothing behind it
  for (int64_t j = t; j <= a.K; j += kVT) {
    int64_t id = -1;
    float lp = 0.0f;
    if (j <= n) {
      id = j < n ? draft_at(a, b, j) : token;
      lp = M<float>::nan();
      if (id >= 0) {
        const double d = (double)load_entry<Tag>(target_row<Tag>(a, b, j), id) - (double)rows[j].m;
        lp = (float)((d * a.c - log2(rows[j].s)) * 0.69314718055994530942);
      }
    }
    a.token_out[b * (a.K + 1) + j] = id;
    a.logp_out[b * (a.K + 1) + j] = lp;
  }
  if (t == 0) a.count_out[b] = n;
}

// ---- host ---------------------------------------------------------------------------------

struct VerifyLayout {
  int rows;
  int64_t chunks;
  size_t stat, row, mass, plan, total;
};
inline VerifyLayout verify_layout(int64_t B, int64_t K, int64_t V, bool with_draft) {
  VerifyLayout l;
  l.rows = (int)(K + 1 + (with_draft ? K : 0));
  l.chunks = (V + kChunk - 1) / kChunk;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.stat = take(sizeof(ChunkStat) * (size_t)(B * l.rows * l.chunks));
  l.row = take(sizeof(RowStat) * (size_t)(B * l.rows));
  l.mass = take(sizeof(double) * (size_t)(B * l.chunks));
  l.plan = take(sizeof(Plan) * (size_t)B);
  l.total = at;
  return l;
}

template <class Tag>
int launch_verify(const VerifyArgs& a, const Ws& ws, hipStream_t st) {
  const uint32_t B = (uint32_t)a.B;
  hipLaunchKernelGGL(verify_stats_kernel<Tag>, dim3(B * a.rows * a.chunks), dim3(kVT), 0, st, a, ws);
  if (int rc = check_launch("verify_stats_kernel")) return rc;
  hipLaunchKernelGGL(verify_decide_kernel<Tag>, dim3(B), dim3(kVT), 0, st, a, ws);
  if (int rc = check_launch("verify_decide_kernel")) return rc;
  if (!a.greedy) {
    hipLaunchKernelGGL(verify_rest_kernel<Tag>, dim3(B * a.chunks), dim3(kVT), 0, st, a, ws);
    if (int rc = check_launch("verify_rest_kernel")) return rc;
  }
  hipLaunchKernelGGL(verify_draw_kernel<Tag>, dim3(B), dim3(kVT), 0, st, a, ws);
  return check_launch("verify_draw_kernel");
}

// Sizes whose index arithmetic and grids fit (a grid's threads are counted in 32 bits).
inline bool verify_fits(int64_t B, int64_t K, int64_t V) {
  if (B < 0 || K < 0 || V < 1 || B > (1 << 20) || K > (1 << 16) || V > ((int64_t)1 << 31) - kChunk)
    return false;
  const int64_t chunks = (V + kChunk - 1) / kChunk;
  return B * (2 * K + 1) <= (((int64_t)1 << 32) / kVT - 1) / chunks;
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" size_t rrl_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V,
                                                    int32_t with_draft_logits) {
  if (!verify_fits(B, K, V)) return 0;
  return verify_layout(B, K, V, with_draft_logits != 0).total;
}

extern "C" int rrl_verify_drafts(const void* target, const void* draft, int32_t dtype, int64_t B,
                                 int64_t K, int64_t V, int64_t t_sb, int64_t t_sk, int64_t d_sb,
                                 int64_t d_sk, rrl_view drafts, const float* uniforms,
                                 double temperature, int32_t do_sample, int64_t* token_out,
                                 int64_t* count_out, float* logp_out, void* workspace,
                                 void* stream) {
  clear_error();
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              "rrl_verify_drafts: logits must be float32, bfloat16 or float16");
  RRL_REQUIRE(B >= 0 && K >= 0, RRL_EINVAL, "rrl_verify_drafts: negative size");
  if (B == 0) return RRL_OK;
  RRL_REQUIRE(V >= 1, RRL_EINVAL, "rrl_verify_drafts: logits need at least one vocabulary entry");
  RRL_REQUIRE(verify_fits(B, K, V), RRL_EINVAL,
              "rrl_verify_drafts: too large (rows * chunks of 4096 entries below 2^24)");
  RRL_REQUIRE(temperature == temperature && temperature < HUGE_VAL, RRL_EINVAL,
              "rrl_verify_drafts: the temperature must be a finite number");
  const bool greedy = !do_sample || temperature <= 0.0;
  RRL_REQUIRE(target != nullptr && token_out != nullptr && count_out != nullptr &&
                  logp_out != nullptr && workspace != nullptr && (K == 0 || drafts.ptr != nullptr) &&
                  (greedy || uniforms != nullptr),
              RRL_EINVAL, "rrl_verify_drafts: null operand");
  RRL_REQUIRE(K == 0 || drafts.dtype == RRL_I32 || drafts.dtype == RRL_I64, RRL_EDTYPE,
              "rrl_verify_drafts: draft tokens must be int32 or int64");
  const size_t size = dtype_size(dtype);
  RRL_REQUIRE((uintptr_t)target % size == 0 && (uintptr_t)draft % size == 0 &&
                  (uintptr_t)uniforms % 4 == 0 && (uintptr_t)workspace % 16 == 0 &&
                  (K == 0 || (uintptr_t)drafts.ptr % dtype_size(drafts.dtype) == 0),
              RRL_EALIGN, "rrl_verify_drafts: a pointer is not aligned to its element");
  if (greedy) draft = nullptr;
  const VerifyLayout l = verify_layout(B, K, V, draft != nullptr);
  VerifyArgs a;
  a.x = static_cast<const char*>(target);
  a.y = K > 0 ? static_cast<const char*>(draft) : nullptr;
  a.xs_b = t_sb;
  a.xs_k = t_sk;
  a.ys_b = d_sb;
  a.ys_k = d_sk;
  a.drafts = drafts.ptr;
  a.drafts_dt = drafts.dtype;
  a.ds_b = drafts.s_row;
  a.ds_k = drafts.s_col;
  a.u = uniforms;
  a.B = B;
  a.K = K;
  a.V = V;
  // a temperature under 1e-290 has the distribution's limit already
  const double t = greedy ? 1.0 : (temperature < 1e-290 ? 1e-290 : temperature);
  a.c = 1.4426950408889634074 / t;
  a.greedy = greedy;
  a.rows = l.rows;
  a.chunks = (int)l.chunks;
  a.token_out = token_out;
  a.count_out = count_out;
  a.logp_out = logp_out;
  char* w = static_cast<char*>(workspace);
  const Ws ws{reinterpret_cast<ChunkStat*>(w + l.stat), reinterpret_cast<RowStat*>(w + l.row),
              reinterpret_cast<double*>(w + l.mass), reinterpret_cast<Plan*>(w + l.plan)};
  hipStream_t st = as_stream(stream);
  if (dtype == RRL_F32) return launch_verify<TagF32>(a, ws, st);
  if (dtype == RRL_BF16) return launch_verify<TagBF16>(a, ws, st);
  return launch_verify<TagF16>(a, ws, st);
}
