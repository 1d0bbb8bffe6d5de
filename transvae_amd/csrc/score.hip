// Log probabilities of given tokens, entropies and most likely alternatives of rows of logits, and their gradient.
//
// One pass over a row: every lane keeps a running maximum m, l = sum exp(x - m) and t = sum exp(x - m) (x - m), rescaled when
// its maximum grows; then with M the row's maximum   ln p_y = x_y - M - ln l,   H = ln l - t / l.
// (t is taken relative to the maximum: sum p x would cancel against ln-sum-exp when all logits are far from zero.)
// The alternatives ride along: a wave keeps its best `top` as a list sorted across its lanes and looks at a vector of logits
// again only if it holds something above the list's last entry, which soon is rare: a row of V values in any random order
// enters top * (1 + ln(V / top)) values a wave.
#include "common.h"

namespace {

struct F16 { _Float16 v; };
struct B16 { uint16_t v; };
constexpr float LOG2E = 1.44269504088896341f;
constexpr int NO_KEY = INT32_MIN;                          // below every value
constexpr int64_t MAX_BLOCKS = (1 << 22) - 1;              // of up to 1024 threads: a grid counts its threads in 32 bits

__device__ inline float value_of(float x) { return x; }
__device__ inline float value_of(B16 x) { return __uint_as_float((uint32_t)x.v << 16); }
__device__ inline float value_of(F16 x) { return (float)x.v; }
__device__ inline void put(float* p, float x) { *p = x; }
__device__ inline void put(F16* p, float x) { p->v = (_Float16)x; }
__device__ inline void put(B16* p, float x) {              // round to nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(x);
  p->v = (u & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

// order of the alternatives as whole numbers: -0 equals +0, NaN is above everything
__device__ inline int key_of(float x) {
  if (x != x) return INT32_MAX;
  const int u = __float_as_int(x + 0.f);
  return u < 0 ? u ^ 0x7FFFFFFF : u;
}
__device__ inline float of_key(int k) { return k == INT32_MAX ? __int_as_float(0x7FC00000) : __int_as_float(k < 0 ? k ^ 0x7FFFFFFF : k); }

struct Sums {
  float m = -INFINITY, l = 0.f, t = 0.f;
  __device__ inline void grow(float to) {                  // to > m
    if (l != 0.f) {                                        // also a NaN
      const float d = m - to, r = __builtin_amdgcn_exp2f(d * LOG2E);
      t = r * (t + l * fmaxf(d, -1e30f));
      l *= r;
    }
    m = to;
  }
  __device__ inline void add(float x) {                    // m is at least x, or x is NaN
    const float d = x - (m == -INFINITY ? 0.f : m), e = __builtin_amdgcn_exp2f(d * LOG2E);
    l += e;
    t = fmaf(e, fmaxf(d, -1e30f), t);                      // -inf adds 0, not 0 * inf
  }
  __device__ inline void join(float m2, float l2, float t2) {
    if (m2 > m) grow(m2);
    if (l2 != 0.f) {
      const float d = m2 - (m == -INFINITY ? 0.f : m), r = __builtin_amdgcn_exp2f(d * LOG2E);
      l += r * l2;
      t += r * (t2 + l2 * fmaxf(d, -1e30f));
    }
  }
};

struct TopList {                                           // lane i < top holds the i-th best
  int key = NO_KEY, idx = 0, last = NO_KEY;                // last: key of entry top - 1, the same in all lanes
  float bar = __int_as_float(0x7FC00000);                  // its value; NaN while the list is not full: nothing is <= NaN
  __device__ inline void insert(int k, int i, int lane, int top) {      // k, i uniform; values come in ascending order of i
    if (k <= last) return;
    const int pos = __popcll(__ballot(lane < top && key >= k));
    const int ku = __shfl_up(key, 1, 64), iu = __shfl_up(idx, 1, 64);
    if (lane > pos) { key = ku; idx = iu; }
    if (lane == pos) { key = k; idx = i; }
    last = __builtin_amdgcn_readlane(key, top - 1);
    bar = last == NO_KEY ? __int_as_float(0x7FC00000) : of_key(last);
  }
};

struct ScoreArgs {
  const void* logits;
  const int64_t* tokens;
  float *logp, *entropy, *stat, *top_logp, *ws;
  int64_t* top_ids;
  int64_t ld, ld_tok, tok_sub, rows, V, ld_logp, ld_ent, seg_len;
  int top, segs;
};

// what is known of a whole row -> its results.  cand: n (key, idx) pairs in shared memory, of which the best `top` are taken.
template <typename T>
__device__ inline void finish_row(const ScoreArgs& a, int64_t row, const Sums& s, const int2* cand, int n, int tid, int threads) {
  const float L = logf(s.l);
  const bool none = s.l == 0.f;                            // -inf everywhere
  if (tid == 0) {
    const int64_t y = a.tokens ? a.tokens[row * a.ld_tok] - a.tok_sub : -1;
    float lp = 0.f;
    if (y >= 0 && y < a.V) lp = none ? -INFINITY : value_of(reinterpret_cast<const T*>(a.logits)[row * a.ld + y]) - s.m - L;
    if (s.l != s.l && y >= 0 && y < a.V) lp = s.l;
    a.logp[row * a.ld_logp] = lp;
    a.entropy[row * a.ld_ent] = none ? 0.f : L - s.t / s.l;
    a.stat[2 * row] = s.m;
    a.stat[2 * row + 1] = L;
  }
  for (int c = tid; c < n; c += threads) {
    const int2 me = cand[c];
    if (me.x == NO_KEY) continue;
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += cand[o].x > me.x || (cand[o].x == me.x && cand[o].y < me.y);
    if (rank < a.top) {
      a.top_ids[row * a.top + rank] = me.y;
      a.top_logp[row * a.top + rank] = none ? -INFINITY : s.l != s.l ? s.l : of_key(me.x) - s.m - L;
    }
  }
}

// W waves share a row (or one part of it); W == 1: a block has four rows.
template <typename T, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void score_kernel(ScoreArgs a) {
  constexpr int NV = Vec<T>::N;
  __shared__ float sums[W == 1 ? 4 : W][3];
  __shared__ int2 cand[W == 1 ? 4 : W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const int kw = W == 1 ? 0 : wave;
  const bool live = row < a.rows;
  const int seg = blockIdx.y;
  Sums s;
  TopList top;
  if (live) {
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
    const int64_t c0 = seg * a.seg_len < a.V ? seg * a.seg_len : a.V, c1 = c0 + a.seg_len < a.V ? c0 + a.seg_len : a.V;
    int64_t head = ((16 - ((uintptr_t)(x + c0) & 15)) & 15) / sizeof(T);              // values up to a 16-byte border
    if (head > c1 - c0) head = c1 - c0;
    const int64_t body = (c1 - c0 - head) / NV, tail = c0 + head + body * NV;
    auto single = [&](int64_t c, bool in) {                // one value a lane
      const float v = in ? value_of(x[c]) : -INFINITY;
      if (in) {
        if (v > s.m) s.grow(v);
        s.add(v);
      }
      if (a.top) {
        uint64_t todo = __ballot(in);
        while (todo) {
          const int o = __ffsll((unsigned long long)todo) - 1;
          todo &= todo - 1;
          top.insert(__builtin_amdgcn_readlane(key_of(v), o), (int)__builtin_amdgcn_readlane((int)c, o), lane, a.top);
        }
      }
    };
    if (kw == 0 && head) single(c0 + lane, lane < head);
    const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + c0 + head);
    for (int64_t i0 = (int64_t)kw * 64; i0 < body; i0 += (int64_t)W * 64) {
      const bool in = i0 + lane < body;
      float v[NV];
      float vm = -INFINITY;
      if (in) {
        const uint4 raw = *reinterpret_cast<const uint4*>(xv + i0 + lane);
        Vec<T> t;
        *reinterpret_cast<uint4*>(t.x) = raw;
#pragma unroll
        for (int e = 0; e < NV; ++e) {
          v[e] = value_of(t.x[e]);
          vm = fmaxf(vm, v[e]);
        }
        if (vm > s.m) s.grow(vm);
#pragma unroll
        for (int e = 0; e < NV; ++e) s.add(v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < NV; ++e) v[e] = 0.f;
      }
      if (a.top) {
        uint64_t todo = __ballot(in && (!(vm <= top.bar) || s.l != s.l));
        while (todo) {                                     // in ascending order of the classes
          const int o = __ffsll((unsigned long long)todo) - 1;
#pragma unroll
          for (int e = 0; e < NV; ++e)
            top.insert(__builtin_amdgcn_readlane(key_of(v[e]), o), (int)(c0 + head + (i0 + o) * NV) + e, lane, a.top);
          todo &= todo - 1;
          todo &= __ballot(in && (!(vm <= top.bar) || s.l != s.l));
        }
      }
    }
    if (kw == 0 && tail < c1) single(tail + lane, tail + lane < c1);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(s.m, o, 64), l2 = __shfl_xor(s.l, o, 64), t2 = __shfl_xor(s.t, o, 64);
    s.join(m2, l2, t2);
  }
  if (lane == 0) { sums[wave][0] = s.m; sums[wave][1] = s.l; sums[wave][2] = s.t; }
  if (lane < a.top) cand[W == 1 ? wave : 0][W == 1 ? lane : wave * a.top + lane] = make_int2(top.key, top.idx);
  __syncthreads();
  if (!live) return;
  Sums all;
  if (W == 1) {
    all.m = sums[wave][0]; all.l = sums[wave][1]; all.t = sums[wave][2];
  } else {
    for (int w = 0; w < W; ++w) all.join(sums[w][0], sums[w][1], sums[w][2]);
  }
  const int n = W == 1 ? a.top : W * a.top, tid = W == 1 ? lane : (int)threadIdx.x, threads = W == 1 ? 64 : 64 * W;
  const int2* c = cand[W == 1 ? wave : 0];
  if (a.segs == 1) {
    finish_row<T>(a, row, all, c, n, tid, threads);
    return;
  }
  float* part = a.ws + (row * a.segs + seg) * (3 + 2 * a.top);          // {m, l, t}, then the part's best (key, idx)
  if (tid == 0) { part[0] = all.m; part[1] = all.l; part[2] = all.t; }
  int* best = reinterpret_cast<int*>(part + 3);
  for (int i = tid; i < a.top; i += threads) { best[2 * i] = NO_KEY; best[2 * i + 1] = 0; }
  __syncthreads();                                                      // W > 1 whenever segs > 1: the whole block is here
  for (int i = tid; i < n; i += threads) {
    const int2 me = c[i];
    if (me.x == NO_KEY) continue;
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += c[o].x > me.x || (c[o].x == me.x && c[o].y < me.y);
    if (rank < a.top) { best[2 * rank] = me.x; best[2 * rank + 1] = me.y; }
  }
}

// joins the parts of a row: a block a row; the parts' lists are merged 16 at a time through shared memory
template <typename T>
__global__ __launch_bounds__(256) void score_join_kernel(ScoreArgs a) {
  __shared__ int2 cand[17 * 64], next[64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, rec = 3 + 2 * a.top;
  const float* part = a.ws + row * a.segs * rec;
  Sums s;
  for (int g = 0; g < a.segs; ++g) s.join(part[(int64_t)g * rec], part[(int64_t)g * rec + 1], part[(int64_t)g * rec + 2]);
  int have = 0;
  for (int g0 = 0; g0 < a.segs && a.top; g0 += 16) {
    const int more = (a.segs - g0 < 16 ? a.segs - g0 : 16) * a.top, n = have + more;
    for (int i = tid; i < more; i += 256) {
      const int* p = reinterpret_cast<const int*>(part + (int64_t)(g0 + i / a.top) * rec + 3) + 2 * (i % a.top);
      cand[have + i] = make_int2(p[0], p[1]);
    }
    __syncthreads();
    if (g0 + 16 >= a.segs) {
      have = n;
      break;
    }
    if (tid < a.top) next[tid] = make_int2(NO_KEY, 0);
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
      const int2 me = cand[i];
      if (me.x == NO_KEY) continue;
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += cand[o].x > me.x || (cand[o].x == me.x && cand[o].y < me.y);
      if (rank < a.top) next[rank] = me;
    }
    __syncthreads();
    if (tid < a.top) cand[tid] = next[tid];
    have = a.top;
    __syncthreads();
  }
  finish_row<T>(a, row, s, cand, have, tid, 256);
}

// ------------------------------------------------------------------------------------------------ gradient
struct ScoreBwdArgs {
  const void* logits;
  void* dx;
  const int64_t *tokens, *top_ids;
  const float *stat, *entropy, *g_logp, *g_entropy, *g_top;
  int64_t ld, ld_tok, tok_sub, rows, V, ld_ent, seg_len;
  int top;
};

// One read and one write a value: p = exp((x - M) - L), dx = -p (pull + g_H (ln p + H)) with pull = g_l + sum g_t; the few
// classes that are the token or an alternative get their own gradient on top, added by the thread that holds the class.
template <typename T>
__global__ __launch_bounds__(256) void score_bwd_kernel(ScoreBwdArgs a) {
  constexpr int NV = Vec<T>::N;
  __shared__ float extra[65];
  __shared__ int64_t which[65];
  __shared__ float pull_s;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t c0 = (int64_t)blockIdx.y * a.seg_len, c1 = c0 + a.seg_len < a.V ? c0 + a.seg_len : a.V;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.V;
  if (tid < 64) {
    int64_t y = a.tokens && a.g_logp ? a.tokens[row * a.ld_tok] - a.tok_sub : -1;
    if (y >= a.V) y = -1;
    const float gl = y >= 0 ? a.g_logp[row] : 0.f;
    const bool alt = a.g_top && tid < a.top;
    const float gt = alt ? a.g_top[row * a.top + tid] : 0.f;
    const int64_t id = alt ? a.top_ids[row * a.top + tid] : -1;
    const bool same = alt && id == y;                                   // the token is an alternative too
    if (tid < 64) { which[1 + tid] = id; extra[1 + tid] = gt + (same ? gl : 0.f); }
    const bool any = __ballot(same) != 0;
    const float sum = wave_sum(gt);
    if (tid == 0) { which[0] = any ? -1 : y; extra[0] = gl; pull_s = gl + sum; }
  }
  __syncthreads();
  const float pull = pull_s, M = a.stat[2 * row], L = a.stat[2 * row + 1], H = a.entropy[row * a.ld_ent];
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const bool none = M == -INFINITY && L == -INFINITY;                   // a row of -inf: no gradient
  auto grad = [&](float v) {
    const float lp = (v - M) - L;
    const float p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float r = -p * (pull + gh * (fmaxf(lp, -1e30f) + H));
    return none || v == -INFINITY ? 0.f : r;
  };
  int64_t head = ((16 - ((uintptr_t)(x + c0) & 15)) & 15) / sizeof(T);
  if (head > c1 - c0) head = c1 - c0;
  const int64_t body = (c1 - c0 - head) / NV, tail = c0 + head + body * NV;
  const bool even = (((uintptr_t)(dx + c0 + head)) & 15) == 0;          // rows of x and dx on the same 16-byte phase
  for (int64_t c = c0 + tid; c < c0 + head; c += 256) put(dx + c, grad(value_of(x[c])));
  for (int64_t i = tid; i < body; i += 256) {
    Vec<T> t;
    *reinterpret_cast<uint4*>(t.x) = *reinterpret_cast<const uint4*>(x + c0 + head + i * NV);
#pragma unroll
    for (int e = 0; e < NV; ++e) put(&t.x[e], grad(value_of(t.x[e])));
    T* d = dx + c0 + head + i * NV;
    if (even) {
      *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(t.x);
    } else {
#pragma unroll
      for (int e = 0; e < NV; ++e) d[e] = t.x[e];
    }
  }
  for (int64_t c = tail + tid; c < c1; c += 256) put(dx + c, grad(value_of(x[c])));
  __syncthreads();                                                      // the rewrites below come after the stores above
  if (tid < 65 && tid <= a.top) {
    const int64_t c = which[tid];
    if (c >= c0 && c < c1) {
      const float v = value_of(x[c]);
      if (!none && v != -INFINITY) put(dx + c, grad(v) + extra[tid]);
    }
  }
}

int type_bytes(int dtype) { return dtype == TVAE_F32 ? 4 : dtype == TVAE_BF16 || dtype == TVAE_F16 ? 2 : 0; }

template <typename T>
void launch_score(const ScoreArgs& a, hipStream_t s) {
  if (a.segs == 1 && a.V <= 2048)
    hipLaunchKernelGGL((score_kernel<T, 1>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((score_kernel<T, 4>), dim3((unsigned)a.rows, a.segs), dim3(256), 0, s, a);
  if (a.segs > 1) hipLaunchKernelGGL((score_join_kernel<T>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
}

}  // namespace

extern "C" int tvae_token_logp(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t ld_tok, int64_t tok_sub,
                               int64_t rows, int64_t V, int top, float* logp, int64_t ld_logp, float* entropy, int64_t ld_ent,
                               float* stat, float* top_logp, int64_t* top_ids, int segs, float* ws, void* stream) {
  TVAE_CHECK(rows >= 0 && V >= 1 && V <= INT32_MAX && ld >= V && top >= 0 && top <= 64 && top <= V, TVAE_E_SHAPE,
             "tvae_token_logp: need rows >= 0, 1 <= V <= ld, top in [0, min(V, 64)] (rows=%lld V=%lld ld=%lld top=%d)", (long long)rows,
             (long long)V, (long long)ld, top);
  TVAE_CHECK(type_bytes(dtype), TVAE_E_DTYPE, "tvae_token_logp: dtype %d is not TVAE_F32, TVAE_BF16 or TVAE_F16", dtype);
  if (rows == 0) return TVAE_OK;
  TVAE_CHECK(logits && logp && entropy && stat && (top == 0 || (top_logp && top_ids)), TVAE_E_NULL, "tvae_token_logp: null pointer");
  TVAE_CHECK((uintptr_t)logits % type_bytes(dtype) == 0, TVAE_E_SHAPE, "tvae_token_logp: logits are not aligned to their type");
  TVAE_CHECK(segs >= 1 && segs <= 1024 && (segs == 1 || ws), TVAE_E_SHAPE, "tvae_token_logp: 1 .. 1024 parts, more than one with a workspace");
  TVAE_CHECK(rows <= MAX_BLOCKS, TVAE_E_SHAPE, "tvae_token_logp: too many rows in one call (%lld)", (long long)rows);
  const int64_t seg_len = ((V + segs - 1) / segs + 7) / 8 * 8;
  ScoreArgs a = {logits, tokens, logp, entropy, stat, top_logp, ws, top_ids, ld, ld_tok, tok_sub, rows, V, ld_logp, ld_ent, seg_len, top, segs};
  if (dtype == TVAE_F32) launch_score<float>(a, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_score<B16>(a, (hipStream_t)stream);
  else launch_score<F16>(a, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_token_logp");
  return TVAE_OK;
}

extern "C" int tvae_token_logp_bwd(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t ld_tok, int64_t tok_sub,
                                   int64_t rows, int64_t V, int top, const float* stat, const float* entropy, int64_t ld_ent,
                                   const int64_t* top_ids, const float* g_logp, const float* g_entropy, const float* g_top, void* dx,
                                   void* stream) {
  TVAE_CHECK(rows >= 0 && V >= 1 && V <= INT32_MAX && ld >= V && top >= 0 && top <= 64 && top <= V, TVAE_E_SHAPE,
             "tvae_token_logp_bwd: need rows >= 0, 1 <= V <= ld, top in [0, min(V, 64)] (rows=%lld V=%lld ld=%lld top=%d)", (long long)rows,
             (long long)V, (long long)ld, top);
  TVAE_CHECK(type_bytes(dtype), TVAE_E_DTYPE, "tvae_token_logp_bwd: dtype %d is not TVAE_F32, TVAE_BF16 or TVAE_F16", dtype);
  if (rows == 0) return TVAE_OK;
  TVAE_CHECK(logits && stat && entropy && dx && (!g_top || top == 0 || top_ids), TVAE_E_NULL, "tvae_token_logp_bwd: null pointer");
  TVAE_CHECK((uintptr_t)logits % type_bytes(dtype) == 0 && (uintptr_t)dx % type_bytes(dtype) == 0, TVAE_E_SHAPE,
             "tvae_token_logp_bwd: logits or dx are not aligned to their type");
  TVAE_CHECK(rows <= MAX_BLOCKS, TVAE_E_SHAPE, "tvae_token_logp_bwd: too many rows in one call (%lld)", (long long)rows);
  const int64_t seg_len = 16384;
  const dim3 grid((unsigned)rows, (unsigned)((V + seg_len - 1) / seg_len));
  TVAE_CHECK(grid.y <= 65535, TVAE_E_SHAPE, "tvae_token_logp_bwd: V too large (%lld)", (long long)V);
  ScoreBwdArgs a = {logits, dx, tokens, top_ids, stat, entropy, g_logp, g_entropy, g_top, ld, ld_tok, tok_sub, rows, V, ld_ent, seg_len,
                    g_top ? top : 0};
  if (dtype == TVAE_F32) hipLaunchKernelGGL(score_bwd_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else if (dtype == TVAE_BF16) hipLaunchKernelGGL(score_bwd_kernel<B16>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(score_bwd_kernel<F16>, grid, dim3(256), 0, (hipStream_t)stream, a);
  TVAE_LAUNCH_CHECK("tvae_token_logp_bwd");
  return TVAE_OK;
}
