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
// are therefore float64, the exponential a polynomial good to 1.1e-12.  An entry takes 12
// float64 instructions and 6 others.  For the 107 M bfloat16 entries of 64 sequences x
// (6 + 5) rows x 151,936 that is 49 us of issue at 2.4 GHz, and their bytes are 45 us at a
// copy's rate; the first launch takes 80 us (2.7 TB/s), for a wave loads its chunk, finds
// the maximum and forms the sum one after another, and only other waves fill its waits.
//
// Rows are cut into chunks, a wave each, so that a single sequence fills the chip:
//   1. verify_stats: the chunks of every row that may be needed: maximum, sum
//   2. verify_rest: joins the rows' chunks and finds n (few sequences: every workgroup
//      for itself, which is shorter than the launch of verify_decide ahead of it),
//      then, after a rejection, the mass of rest in each part of row n
//   3. verify_draw: a workgroup per sequence finds the chunk, then the entry
#include "vocab_weights.hpp"

namespace rrl {
namespace {

constexpr int kVT = 256;        // threads of a workgroup
constexpr int kMass = 1024;     // entries whose rest is summed by a wave

// Weights below this count as none.
constexpr double kNothing = 0x1p-960;

// A probability differs from another by no more than rounding if by less than this of it.
// Each is off by five exponentials' 1.1e-12 (its weight, the factor of its row, and the
// row's sum, whose chunks have a factor and are brought to one maximum), so that equal
// ones lie up to 1.1e-11 apart, however the two rows were shifted or summed.
constexpr double kSame = 0x1p-35;

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
  int chunks, chunk;            // chunks of a row, and a chunk's entries (1024, 2048 or 4096)
  int masses;                   // parts of kMass entries
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
  double* mass;     // [B, masses]
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

// Whether one of the sequence's first `n` drafts is missing; the whole wave takes part.
__device__ __forceinline__ bool draft_ends_before(const VerifyArgs& a, int64_t b, int n) {
  const int lane = threadIdx.x & 63;
  for (int k = 0; k < n; k += 64)
    if (__any(k + lane < n && draft_at(a, b, k + lane) < 0)) return true;
  return false;
}

// ---- 1: chunks -----------------------------------------------------------------------

template <class Tag, int NS, bool DIRECT>
__device__ __forceinline__ double weigh(u32x4 (&raw)[NS], const Weight& weight) {
  constexpr int EPV = Pack16<Tag>::EPV;
  double part[2] = {0.0, 0.0};
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    // unpacked again here, a slab at a time: values kept since the maximum, or more
    // slabs in flight, would take registers that more waves make better use of
    asm volatile("" : "+v"(raw[s]));
    float x[EPV];
    Pack16<Tag>::unpack(raw[s], x);
#pragma unroll
    for (int k = 0; k < EPV; ++k) part[k & 1] += weight.unscaled<DIRECT>(x[k]);
    __builtin_amdgcn_sched_barrier(0);
  }
  return (part[0] + part[1]) * weight.factor<DIRECT>();
}

template <class Tag, int NS>
__global__ __launch_bounds__(kVT) void verify_stats_kernel(VerifyArgs a, Ws ws) {
  constexpr int EPV = Pack16<Tag>::EPV;
  const int lane = threadIdx.x & 63;
  const uint32_t id = __builtin_amdgcn_readfirstlane(blockIdx.x * (kVT / 64) + (threadIdx.x >> 6));
  const uint32_t rid = id / a.chunks, chunk = id % a.chunks;
  const int64_t b = rid / a.rows;
  const int r = (int)(rid % a.rows);
  if (b >= a.B) return;
  // target row j serves only if the j drafts before it exist, draft row j also its own;
  // a row behind the draft's end may not be there to be read, so the drafts come first
  const bool is_draft = r > a.K;
  const int j = is_draft ? r - (int)a.K - 1 : r;
  if (draft_ends_before(a, b, j + (is_draft ? 1 : 0))) return;
  const char* row = is_draft ? draft_row<Tag>(a, b, j) : target_row<Tag>(a, b, j);
  const int64_t lo = (int64_t)chunk * (NS * 64 * EPV) + lane * EPV;
  u32x4 raw[NS];
  if ((int64_t)(chunk + 1) * (NS * 64 * EPV) <= a.V) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
      raw[s] = reinterpret_cast<const Any16*>(row + (lo + s * 64 * EPV) * (16 / EPV))->v;
  } else {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float x[EPV];
      load_entries<Tag>(row, lo + s * 64 * EPV, a.V, x);
      raw[s] = Pack16<Tag>::pack(x);
    }
  }
  float m = -M<float>::inf();
  bool nan = false;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float x[EPV];
    Pack16<Tag>::unpack(raw[s], x);
#pragma unroll
    for (int k = 0; k < EPV; k += 2) {
      // with NaN among them the result is not used
      asm("v_max3_f32 %0, %1, %2, %0" : "+v"(m) : "v"(x[k]), "v"(x[k + 1]));
      nan |= __builtin_isunordered(x[k], x[k + 1]);
    }
  }
  m = wave_max_dpp(m);
  if (__any(nan)) m = M<float>::inf();
  int at = 0x7fffffff;
  double sum = 0.0;
  if (m > -M<float>::inf() && m < M<float>::inf()) {
    const Weight weight(m, a.c, 1.0);
    sum = weight.direct ? weigh<Tag, NS, true>(raw, weight) : weigh<Tag, NS, false>(raw, weight);
    sum = wave_sum_d(sum);
    if (a.greedy) {  // read again: kept, the entries would take registers from sampling
      for (int s = NS - 1; s >= 0; --s) {
        float x[EPV];
        load_entries<Tag>(row, lo + s * 64 * EPV, a.V, x);
#pragma unroll
        for (int k = EPV - 1; k >= 0; --k)
          if (x[k] == m) at = (int)(lo + s * 64 * EPV + k);
      }
      at = wave_min_dpp(at);
    }
  }
  if (lane == 0) ws.stat[id] = ChunkStat{sum, m, at};
}

// ---- 2: rows, how far the draft is accepted, and the rest's chunks ------------------------

// Joins the chunks of one row; 16 lanes take part.  The first kAhead of a lane's
// chunks are loaded together.
__device__ __forceinline__ RowStat join_row(const ChunkStat* st, int chunks, double c) {
  constexpr int kAhead = 10;
  const int lane = threadIdx.x & 15;
  ChunkStat mine[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int i = lane + 16 * k;
    mine[k] = i < chunks ? st[i] : ChunkStat{0.0, -M<float>::inf(), 0x7fffffff};
  }
  float m = -M<float>::inf();
#pragma unroll
  for (int k = 0; k < kAhead; ++k) m = fmaxf(m, mine[k].m);
  for (int i = lane + 16 * kAhead; i < chunks; i += 16) m = fmaxf(m, st[i].m);
  m = row16_max(m);
  if (m == -M<float>::inf()) m = M<float>::inf();  // nothing is possible: no distribution
  double s = 0.0;
  int at = 0x7fffffff;
  auto add = [&](const ChunkStat& v) {
    s += v.s * exp2_neg(((double)v.m - (double)m) * c);
    if (v.m == m) at = min(at, v.at);
  };
  if (m < M<float>::inf()) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) add(mine[k]);
    for (int i = lane + 16 * kAhead; i < chunks; i += 16) add(st[i]);
  }
  return RowStat{row16_sum(s), m, row16_min(at)};
}

// What an entry of the deciding row weighs.
template <class Tag>
struct Rest {
  const char *x, *y;
  Weight p, q;
  int64_t skip;  // an entry without mass (the rejected draft), or -1
  bool direct;
  template <bool DIRECT>
  __device__ __forceinline__ void weights(int64_t i, int64_t V, double (&w)[Pack16<Tag>::EPV]) const {
    constexpr int EPV = Pack16<Tag>::EPV;
    float v[EPV], d[EPV];
    load_entries<Tag>(x, i, V, v);
    if (y) load_entries<Tag>(y, i, V, d);
#pragma unroll
    for (int k = 0; k < EPV; ++k) w[k] = p.template unscaled<DIRECT>(v[k]) * p.template factor<DIRECT>();
    if (y) {
      const double f = q.template factor<DIRECT>();
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        const double rest = fma(-f, q.template unscaled<DIRECT>(d[k]), w[k]);
        w[k] = rest > kSame * w[k] ? rest : 0.0;
      }
    }
#pragma unroll
    for (int k = 0; k < EPV; ++k)
      if (i + k == skip) w[k] = 0.0;
  }
  __device__ __forceinline__ void weights(int64_t i, int64_t V, double (&w)[Pack16<Tag>::EPV]) const {
    if (direct) weights<true>(i, V, w);
    else weights<false>(i, V, w);
  }
};

template <class Tag>
__device__ __forceinline__ Rest<Tag> rest_of(const VerifyArgs& a, const RowStat* row, int64_t b,
                                             int n, int kind) {
  Rest<Tag> r;
  r.x = target_row<Tag>(a, b, n);
  r.y = nullptr;
  r.p = Weight(row[n].m, a.c, 1.0 / row[n].s);
  r.skip = -1;
  r.direct = r.p.direct;
  if (kind == REST_PQ) {
    const RowStat q = row[a.K + 1 + n];
    r.y = draft_row<Tag>(a, b, n);
    r.q = Weight(q.m, a.c, 1.0 / q.s);
    r.direct &= r.q.direct;
  } else if (kind == REST_P_WITHOUT_DRAFT) {
    r.skip = draft_at(a, b, n);
  }
  return r;
}

// What deciding position j takes from its rows, d its draft; beyond the draft's end at
// L, whose rows may not be there, and where d names no entry, only d.
struct Position {
  int64_t d;
  float x, y, u;
};
template <class Tag>
__device__ __forceinline__ Position position(const VerifyArgs& a, int64_t b, int64_t j, int64_t d,
                                             int L) {
  Position p{d, 0.0f, 0.0f, 0.0f};
  if (j >= L || p.d < 0 || p.d >= a.V || a.greedy) return p;
  p.x = load_entry<Tag>(target_row<Tag>(a, b, j), p.d);
  if (a.y) p.y = load_entry<Tag>(draft_row<Tag>(a, b, j), p.d);
  p.u = a.u[b * (a.K + 1) + j];
  return p;
}

// Its verdict: -1 (accepted), or what the next token is drawn from.
__device__ __forceinline__ int judge(const VerifyArgs& a, const RowStat* row, int64_t j,
                                     const Position& at) {
  const RowStat p = row[j];
  if (!(p.m < M<float>::inf()) || at.d >= a.V) return REST_BAD;
  if (a.greedy) return at.d == p.at ? -1 : REST_P;
  double qx = 1.0;
  if (a.y) {
    const RowStat q = row[a.K + 1 + j];
    if (!(q.m < M<float>::inf())) return REST_BAD;
    qx = Weight(q.m, a.c, 1.0 / q.s).one(at.y);
    if (!(qx > kNothing)) qx = 0.0;
  }
  double px = Weight(p.m, a.c, 1.0 / p.s).one(at.x);
  if (!(px > kNothing)) px = 0.0;
  if ((double)at.u * qx < px) return -1;
  return a.y ? REST_PQ : REST_P_WITHOUT_DRAFT;
}

template <class Tag, int NS, bool DIRECT>
__device__ __forceinline__ double rest_sum(const Rest<Tag>& r, int64_t lo, int64_t V) {
  constexpr int EPV = Pack16<Tag>::EPV;
  double sum = 0.0;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    double w[EPV];
    r.template weights<DIRECT>(lo + s * 64 * EPV, V, w);
#pragma unroll
    for (int k = 0; k < EPV; ++k) sum += w[k];
  }
  return sum;
}

constexpr int kRowsHeld = 64;  // rows whose statistics a workgroup keeps in LDS

// Joins the sequence's rows and finds its plan; the whole workgroup takes part.
// The rows' statistics are left in `held`, or, for long drafts, in the workspace,
// where they go also if `write`.
template <class Tag>
__device__ __forceinline__ Plan decide(const VerifyArgs& a, const Ws& ws, int64_t b, bool write,
                                       RowStat* held, const RowStat*& rows) {
  const int t = threadIdx.x, lane = t & 63;
  __shared__ int sh_len, sh_n, sh_rest;
  const int64_t d = t < a.K ? draft_at(a, b, t) : -1;
  if (t < 64) {
    int len = (int)a.K;
    for (int k = 0; k < a.K; k += 64) {
      const uint64_t gone = __ballot(k + lane < a.K && draft_at(a, b, k + lane) < 0);
      if (gone) {
        len = k + __ffsll((unsigned long long)gone) - 1;
        break;
      }
    }
    if (t == 0) {
      sh_len = sh_n = len;
      sh_rest = REST_P;
    }
  }
  __syncthreads();
  const int L = sh_len;
  Position at = position<Tag>(a, b, t, d, L);  // these loads are under way while the rows are joined
  // in the workspace, the groups of a sequence write equal values
  RowStat* row = a.rows <= kRowsHeld ? held : ws.row + b * a.rows;
  rows = row;
  for (int r = t / 16; r < a.rows; r += kVT / 16) {
    const bool is_draft = r > a.K;
    if (is_draft ? r - (int)a.K - 1 >= L : r > L) continue;
    const RowStat s = join_row(ws.stat + (b * a.rows + r) * a.chunks, a.chunks, a.c);
    if ((t & 15) == 0) {
      row[r] = s;
      if (write) ws.row[b * a.rows + r] = s;
    }
  }
  __syncthreads();
  // positions in turn, kVT at a time: the first that does not accept its draft
  for (int j0 = 0; j0 < L && sh_n == L; j0 += kVT) {
    const int j = j0 + t;
    if (j0 > 0) at = position<Tag>(a, b, j, j < L ? draft_at(a, b, j) : -1, L);
    const int rest = j < L ? judge(a, row, j, at) : -1;
    __syncthreads();
    if (rest >= 0) atomicMin(&sh_n, j);
    __syncthreads();
    if (rest >= 0 && sh_n == j) sh_rest = rest;
    __syncthreads();
  }
  Plan pl{sh_n, sh_rest};
  if (pl.n == L && !(row[L].m < M<float>::inf())) pl.rest = REST_BAD;
  if (write && t == 0) ws.plan[b] = pl;
  return pl;
}

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_decide_kernel(VerifyArgs a, Ws ws) {
  __shared__ RowStat held[kRowsHeld];
  const RowStat* row;
  decide<Tag>(a, ws, blockIdx.x, true, held, row);
}

template <class Tag, bool DECIDED>
__global__ __launch_bounds__(kVT) void verify_rest_kernel(VerifyArgs a, Ws ws, int groups) {
  constexpr int EPV = Pack16<Tag>::EPV, NS = kMass / (64 * EPV);
  const int64_t b = blockIdx.x / groups;
  const int group = (int)(blockIdx.x % groups), t = threadIdx.x, lane = t & 63;
  __shared__ RowStat held[DECIDED ? 1 : kRowsHeld];
  const RowStat* row = ws.row + b * a.rows;
  Plan pl;
  if constexpr (DECIDED) pl = ws.plan[b];
  else pl = decide<Tag>(a, ws, b, group == 0, held, row);
  if (pl.rest != REST_PQ && pl.rest != REST_P_WITHOUT_DRAFT) return;
  const Rest<Tag> r = rest_of<Tag>(a, row, b, pl.n, pl.rest);
  for (int part = group * (kVT / 64) + (t >> 6); part < a.masses; part += groups * (kVT / 64)) {
    const int64_t lo = (int64_t)part * kMass + lane * EPV;
    double sum = r.direct ? rest_sum<Tag, NS, true>(r, lo, a.V) : rest_sum<Tag, NS, false>(r, lo, a.V);
    sum = wave_sum_d(sum);
    if (lane == 0) ws.mass[b * a.masses + part] = sum;
  }
}

// ---- 3: the last token -------------------------------------------------------------------

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
// Least value over the workgroup.
__device__ __forceinline__ int block_min(int v, int* sh) {
  v = wave_min_dpp(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return min(min(sh[0], sh[1]), min(sh[2], sh[3]));
}

template <class Tag>
__global__ __launch_bounds__(kVT) void verify_draw_kernel(VerifyArgs a, Ws ws) {
  constexpr int EPV = Pack16<Tag>::EPV;
  constexpr int kNone = 0x7fffffff;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  const Plan pl = ws.plan[b];
  const int n = pl.n;
  const RowStat* rows = ws.row + b * a.rows;
  __shared__ double sh[kVT / 64];
  __shared__ int shi[kVT / 64];
  __shared__ double sh_rem;
  int64_t token = -1;
  if (pl.rest != REST_BAD && a.greedy) {
    token = rows[n].at;
  } else if (pl.rest != REST_BAD) {
    const double u = a.u[b * (a.K + 1) + a.K];
    const ChunkStat* st = ws.stat + (b * a.rows + n) * a.chunks;
    const RowStat p = rows[n];
    int kind = pl.rest, parts, size;
    auto part_mass = [&](int k) {
      if (k >= parts) return 0.0;
      if (kind != REST_P) return ws.mass[b * a.masses + k];
      return st[k].s * exp2_neg(((double)st[k].m - (double)p.m) * a.c) / p.s;
    };
    auto whole_mass = [&]() {
      parts = kind != REST_P ? a.masses : a.chunks;
      size = kind != REST_P ? kMass : a.chunk;
      double v = 0.0, total;
      for (int k = t; k < parts; k += kVT) v += part_mass(k);
      block_scan(v, total, sh);
      return total;
    };
    double total = whole_mass();
    if (!(total > kNothing)) {  // the two rows are equal to within rounding
      kind = REST_P;
      total = whole_mass();
    }
    // the first part whose running sum passes the border, else the last with any mass
    const double border = u * total;
    double before = 0.0;
    int chunk = kNone, last = kNone;  // last: negated
    for (int k0 = 0; k0 < parts && chunk == kNone; k0 += kVT) {
      const double w = part_mass(k0 + t);
      double sum;
      const double incl = block_scan(w, sum, sh) + before;
      chunk = block_min(w > kNothing && incl > border ? k0 + t : kNone, shi);
      last = min(last, block_min(w > kNothing ? -(k0 + t) : kNone, shi));
      if (chunk == k0 + t) sh_rem = border - (incl - w);
      before += sum;
    }
    __syncthreads();
    const bool over = chunk == kNone;
    // (parts whose every mass counts as none, though their sum does not: the first)
    if (over) chunk = last != kNone ? -last : 0;
    const double rem = over ? M<double>::inf() : sh_rem;
    const Rest<Tag> r = rest_of<Tag>(a, rows, b, n, kind);
    int first = kNone;
    last = kNone;
    before = 0.0;
    for (int e = 0; e < size; e += kVT * EPV) {
      const int e0 = e + t * EPV;
      double w[EPV] = {}, mine = 0.0, sum;
      if (e0 < size) r.weights((int64_t)chunk * size + e0, a.V, w);
#pragma unroll
      for (int k = 0; k < EPV; ++k) mine += w[k];
      double at = block_scan(mine, sum, sh) - mine + before;
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        at += w[k];
        if (w[k] > kNothing) {
          last = min(last, -(e0 + k));
          if (at > rem) first = min(first, e0 + k);
        }
      }
      before += sum;
    }
    first = block_min(first, shi);
    last = block_min(last, shi);
    token = (int64_t)chunk * size + (first != kNone ? first : (last != kNone ? -last : 0));
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
        // the sum, at least 1, may come out 1e-12 under it where one entry holds all mass
        lp = fminf((float)((d * a.c - log2(rows[j].s)) * 0.69314718055994530942), 0.0f);
      }
    }
    a.token_out[b * (a.K + 1) + j] = id;
    a.logp_out[b * (a.K + 1) + j] = lp;
  }
  if (t == 0) a.count_out[b] = n;
}

// ---- host ---------------------------------------------------------------------------------

// Entries of a chunk: as many as leave the 1024 SIMDs enough waves to hide loads
// behind, for a longer chunk spends less on its sum.  A call took, in us with 1024 / 2048 /
// 4096 entries, by its chunks of 1024:
//   5 drafts of 151,936 bfloat16: 6,556 25.0 / 25.2 / 26.6, 14,751 32.7 / 31.8 / 33.1,
//   18,029 35.3 / 34.5 / 35.4, 39,336 54.2 / 51.2 / 51.5, 42,614 56.9 / 53.2 / 53.8,
//   78,672 91.1 / 82.7 / 81.3;
//   3 drafts of 50,257 float32: 14,000 31.1 / 32.4 / 36.9, 21,000 38.2 / 38.5 / 43.7,
//   38,500 57.2 / 54.8 / 59.7, 45,500 64.0 / 60.6 / 65.6 (the second border is early here).
constexpr int64_t kMost1024 = 16384, kMost2048 = 40960;
inline int chunk_entries(int64_t rows, int64_t V) {
  const int64_t least = rows * ((V + 1023) / 1024);
  return least <= kMost1024 ? 1024 : (least <= kMost2048 ? 2048 : 4096);
}

// Chunks of `rows` rows or of any smaller number of them, of which there may be more, for
// they may be shorter: a workspace serves every smaller batch, shorter draft, and a call
// that leaves the draft logits out (greedy decoding among them).
inline int64_t chunks_at_most(int64_t rows, int64_t V) {
  const int64_t c1 = (V + 1023) / 1024, c2 = (V + 2047) / 2048, c4 = (V + 4095) / 4096;
  const int64_t with_c1 = kMost1024 / c1, with_c2 = kMost2048 / c1;  // rows in chunks of 1024, 2048
  return max(rows * c4, max(min(rows, with_c1) * c1, min(rows, with_c2) * c2));
}

struct VerifyLayout {
  int rows, chunk;
  int64_t chunks, masses;
  size_t stat, row, mass, plan, total;
};
inline VerifyLayout verify_layout(int64_t B, int64_t K, int64_t V, bool with_draft) {
  VerifyLayout l;
  l.rows = (int)(K + 1 + (with_draft ? K : 0));
  l.chunk = chunk_entries(B * l.rows, V);
  l.chunks = (V + l.chunk - 1) / l.chunk;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.stat = take(sizeof(ChunkStat) * (size_t)chunks_at_most(B * l.rows, V));
  l.row = take(sizeof(RowStat) * (size_t)(B * l.rows));
  l.masses = (V + kMass - 1) / kMass;
  l.mass = take(sizeof(double) * (size_t)(B * l.masses));
  l.plan = take(sizeof(Plan) * (size_t)B);
  l.total = at;
  return l;
}

template <class Tag, int CHUNK>
int launch_verify(const VerifyArgs& a, const Ws& ws, hipStream_t st) {
  constexpr int kWaves = kVT / 64, NS = CHUNK / (64 * Pack16<Tag>::EPV);
  const uint32_t B = (uint32_t)a.B, waves = B * a.rows * a.chunks;
  const uint32_t groups = (uint32_t)(a.masses + kWaves - 1) / kWaves;
  hipLaunchKernelGGL((verify_stats_kernel<Tag, NS>), dim3((waves + kWaves - 1) / kWaves), dim3(kVT), 0,
                     st, a, ws);
  if (int rc = check_launch("verify_stats_kernel")) return rc;
  if (a.greedy || B * groups > 1024) {  // more workgroups than run at once
    hipLaunchKernelGGL(verify_decide_kernel<Tag>, dim3(B), dim3(kVT), 0, st, a, ws);
    if (int rc = check_launch("verify_decide_kernel")) return rc;
    if (!a.greedy)
      hipLaunchKernelGGL((verify_rest_kernel<Tag, true>), dim3(B * groups), dim3(kVT), 0, st, a, ws,
                         (int)groups);
  } else {
    hipLaunchKernelGGL((verify_rest_kernel<Tag, false>), dim3(B * groups), dim3(kVT), 0, st, a, ws,
                       (int)groups);
  }
  if (int rc = check_launch("verify_rest_kernel")) return rc;
  hipLaunchKernelGGL(verify_draw_kernel<Tag>, dim3(B), dim3(kVT), 0, st, a, ws);
  return check_launch("verify_draw_kernel");
}
template <class Tag>
int launch_verify(const VerifyArgs& a, const Ws& ws, hipStream_t st) {
  if (a.chunk == 1024) return launch_verify<Tag, 1024>(a, ws, st);
  if (a.chunk == 2048) return launch_verify<Tag, 2048>(a, ws, st);
  return launch_verify<Tag, 4096>(a, ws, st);
}

// Sizes whose index arithmetic and grids fit (a grid's threads are counted in 32 bits).
inline bool verify_fits(int64_t B, int64_t K, int64_t V) {
  if (B < 0 || K < 0 || V < 1 || B > (1 << 20) || K > (1 << 16) || V > ((int64_t)1 << 31) - 4096)
    return false;
  return B * (2 * K + 1) <= ((int64_t)1 << 23) / ((V + 4095) / 4096);
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
              "rrl_verify_drafts: too large (over 2^23 chunks of 4096 entries)");
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
  a.chunk = l.chunk;
  a.masses = (int)l.masses;
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
