// Layer norm with weight and bias, forward (with the statistics that its gradient needs) and backward.
//
//   forward    u = (x - mean) rstd,  y = u w + b            mean, rstd = 1 / sqrt(var + eps) of each row, fp32
//   backward   g = dy w,  dx = rstd (g - mean_c(g) - u mean_c(g u)),  dw = sum_rows dy u,  db = sum_rows dy
//
// Both are bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx, once each.
// A row belongs to a team of threads and lives in its registers between the load and the store: part of a warp for
// narrow rows, one to sixteen warps (at most 16 values a thread) for wide ones.  A team goes through many rows, and a
// thread always has the same columns: weight and bias stay in its registers, and so do its columns' sums for dw and
// db, which leave the SM once (one partial row per CTA, added up by a second kernel in a fixed order: no atomics, the
// same bits every time).  The next row is requested before the current one is reduced.  A row takes one barrier:
// the forward's warps form their own mean and squared deviations and merge both,
//   M2 = sum_w M2_w + sum_w n_w (mean_w - mean)^2,
// the backward's two sums are known in one pass.
#include "kernels.h"
#include "ptx.cuh"

namespace sd3 {

int device_sm_count();

namespace {

constexpr int LNB_THREADS = 512;   // at most, of a CTA
constexpr int LNB_PER_THREAD = 16; // values of a row that a thread holds, at most
constexpr int LNB_MAX_C = LNB_THREADS * LNB_PER_THREAD;  // wider rows: the kernels at the end of this file
constexpr int LNB_MAX_WARPS = LNB_THREADS / 32;

// VEC values of type T as they lie in memory: 16 bytes, or one value where rows are not 16-byte aligned
template <typename T, int VEC>
struct Raw;
template <>
struct Raw<bf16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static void store(bf16* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  __device__ __forceinline__ static void store(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_float(bf16* p, float v) { *p = __float2bfloat16_rn(v); }
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { from_float(&v, 0.f); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_float(v); }
  __device__ __forceinline__ static void store(T* p, const float (&f)[1]) { from_float(p, f[0]); }
};

__device__ __forceinline__ void team_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// sum over the LANES lanes of a (part of a) warp, the same bits in every lane
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct LnFwdArgs {
  const void* x;
  long ldx;
  const float *w, *b;
  void* y;
  float *mean, *rstd;
  long rows;
  int C, warps, teams;
  float eps;
};

template <typename T, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(LNB_THREADS, 1) layer_norm_kernel(const __grid_constant__ LnFwdArgs a) {
  __shared__ float2 part[2][LNB_MAX_WARPS];  // mean and squared deviations of each warp, two rows' worth
  __shared__ float n_of[LNB_MAX_WARPS];      // values that each warp holds of a row
  grid_dep_wait();
  grid_dep_launch();
  const int ts = a.warps > 1 ? 32 * a.warps : LANES;  // threads of a team
  const int team = threadIdx.x / ts, t = threadIdx.x % ts;
  const int warp0 = team * a.warps;  // the team's first warp (several warps a team)
  const int nvec = a.C / VEC;
  const float inv_c = 1.0f / static_cast<float>(a.C);
  float w[NV][VEC], b[NV][VEC];
  int count = 0;  // values of this thread
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * ts;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = c < nvec && a.w ? a.w[c * VEC + j] : 1.f;
      b[i][j] = c < nvec && a.b ? a.b[c * VEC + j] : 0.f;
    }
    count += c < nvec ? VEC : 0;
  }
  const float n_warp = lanes_sum<LANES>(static_cast<float>(count));
  const float inv_n = n_warp > 0.f ? 1.0f / n_warp : 0.f;
  if ((threadIdx.x & 31) == 0) n_of[threadIdx.x >> 5] = n_warp;  // read after the team's first barrier
  const long step = static_cast<long>(gridDim.x) * a.teams;
  const long first = static_cast<long>(blockIdx.x) * a.teams;
  Raw<T, VEC> next[NV];
  auto request = [&](long row) {
    const T* p = static_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * ts;
      if (row < a.rows && c < nvec) next[i].load(p + c * VEC);
      else next[i].zero();
    }
  };
  request(first + team);
  int buf = 0;
  // `base` is the same for the whole CTA: lanes of one warp may belong to teams with and without a row
  for (long base = first; base < a.rows; base += step) {
    const long row = base + team;
    float v[NV][VEC];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next[i].get(v[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += v[i][j];
    }
    request(row + step);
    float mean = lanes_sum<LANES>(sum) * inv_n;
    float m2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * ts < nvec) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) m2 = fmaf(v[i][j] - mean, v[i][j] - mean, m2);
      }
    m2 = lanes_sum<LANES>(m2);
    if (a.warps > 1) {
      const int warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0) part[buf][warp] = make_float2(mean, m2);
      team_barrier(1 + team, ts);
      float s = 0.f;
      for (int k = 0; k < a.warps; ++k) s = fmaf(part[buf][warp0 + k].x, n_of[warp0 + k], s);
      mean = s * inv_c;
      m2 = 0.f;
      for (int k = 0; k < a.warps; ++k) {
        const float2 p = part[buf][warp0 + k];
        m2 += fmaf((p.x - mean) * (p.x - mean), n_of[warp0 + k], p.y);
      }
      buf ^= 1;
    }
    const float rstd = 1.0f / sqrtf(m2 * inv_c + a.eps);
    if (row < a.rows) {
      T* out = static_cast<T*>(a.y) + row * a.C;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t + i * ts;
        if (c < nvec) {
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = fmaf((v[i][j] - mean) * rstd, w[i][j], b[i][j]);
          Raw<T, VEC>::store(out + c * VEC, o);
        }
      }
      if (t == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
      }
    }
  }
}

struct LnBwdArgs {
  const void* dy;
  long lddy;
  const void* x;
  long ldx;
  const float *w, *mean, *rstd;
  void* dx;
  float* partial;  // (gridDim.x, 2, C): this CTA's share of dw and db
  long rows;
  int C, warps, teams;
};

template <typename T, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(LNB_THREADS, 1) layer_norm_backward_kernel(const __grid_constant__ LnBwdArgs a) {
  extern __shared__ float sums[];  // 2 C: dw and db of this CTA, at the end
  __shared__ float2 part[2][LNB_MAX_WARPS];
  grid_dep_wait();
  grid_dep_launch();
  const int ts = a.warps > 1 ? 32 * a.warps : LANES;
  const int team = threadIdx.x / ts, t = threadIdx.x % ts;
  const int warp0 = team * a.warps;
  const int nvec = a.C / VEC;
  const float inv_c = 1.0f / static_cast<float>(a.C);
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * ts;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = c < nvec && a.w ? a.w[c * VEC + j] : 1.f;
      dw[i][j] = 0.f;
      db[i][j] = 0.f;
    }
  }
  const long step = static_cast<long>(gridDim.x) * a.teams;
  const long first = static_cast<long>(blockIdx.x) * a.teams;
  Raw<T, VEC> nx[NV], ny[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto request = [&](long row) {
    const T* px = static_cast<const T*>(a.x) + row * a.ldx;
    const T* py = static_cast<const T*>(a.dy) + row * a.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * ts;
      if (row < a.rows && c < nvec) {
        nx[i].load(px + c * VEC);
        ny[i].load(py + c * VEC);
      } else {
        nx[i].zero();
        ny[i].zero();
      }
    }
    nmean = row < a.rows ? a.mean[row] : 0.f;
    nrstd = row < a.rows ? a.rstd[row] : 0.f;
  };
  request(first + team);
  int buf = 0;
  for (long base = first; base < a.rows; base += step) {
    const long row = base + team;
    Raw<T, VEC> rx[NV], ry[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) { rx[i] = nx[i]; ry[i] = ny[i]; }
    const float mean = nmean, rstd = nrstd;
    request(row + step);
    // a place without a value has dy = 0 and adds nothing
    float sg = 0.f, sgu = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[VEC], dy[VEC];
      rx[i].get(x);
      ry[i].get(dy);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = (x[j] - mean) * rstd, g = dy[j] * w[i][j];
        sg += g;
        sgu = fmaf(g, u, sgu);
        dw[i][j] = fmaf(dy[j], u, dw[i][j]);
        db[i][j] += dy[j];
      }
    }
    sg = lanes_sum<LANES>(sg);
    sgu = lanes_sum<LANES>(sgu);
    if (a.warps > 1) {
      if ((threadIdx.x & 31) == 0) part[buf][threadIdx.x >> 5] = make_float2(sg, sgu);
      team_barrier(1 + team, ts);
      sg = 0.f;
      sgu = 0.f;
      for (int k = 0; k < a.warps; ++k) {
        sg += part[buf][warp0 + k].x;
        sgu += part[buf][warp0 + k].y;
      }
      buf ^= 1;
    }
    const float mg = sg * inv_c, mgu = sgu * inv_c;
    if (row < a.rows) {
      T* out = static_cast<T*>(a.dx) + row * a.C;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t + i * ts;
        if (c < nvec) {
          float x[VEC], dy[VEC], o[VEC];
          rx[i].get(x);
          ry[i].get(dy);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float u = (x[j] - mean) * rstd;
            o[j] = rstd * (fmaf(dy[j], w[i][j], -mg) - u * mgu);
          }
          Raw<T, VEC>::store(out + c * VEC, o);
        }
      }
    }
  }
  // the teams' sums: those of one warp by shuffles, then one group of threads after the other in shared memory
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], o);
        db[i][j] += __shfl_xor_sync(0xffffffffu, db[i][j], o);
      }
  const int group = a.warps > 1 ? team : static_cast<int>(threadIdx.x >> 5);
  const int groups = a.warps > 1 ? a.teams : static_cast<int>(blockDim.x >> 5);
  const bool mine = a.warps > 1 || (threadIdx.x & 31) < LANES;
  for (int s = 0; s < groups; ++s) {
    if (group == s && mine) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t + i * ts;
        if (c < nvec) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            sums[c * VEC + j] = dw[i][j] + (s > 0 ? sums[c * VEC + j] : 0.f);
            sums[a.C + c * VEC + j] = db[i][j] + (s > 0 ? sums[a.C + c * VEC + j] : 0.f);
          }
        }
      }
    }
    __syncthreads();
  }
  float* out = a.partial + static_cast<long>(blockIdx.x) * 2 * a.C;
  for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) out[c] = sums[c];
}

// dw and db: the sums of `parts` partial rows of 2 C values.  A thread adds every eighth of its column's, then the
// eight threads of a column are added up.
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const float* partial, int parts, int C, float* dw,
                                                                 float* db) {
  __shared__ float s[8][32];
  grid_dep_wait();
  grid_dep_launch();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), k0 = threadIdx.x >> 5;
  float v = 0.f;
  if (col < 2 * C)
    for (int k = k0; k < parts; k += 8) v += partial[static_cast<long>(k) * 2 * C + col];
  s[k0][threadIdx.x & 31] = v;
  __syncthreads();
  if (k0 == 0 && col < 2 * C) {
    float r = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) r += s[k][threadIdx.x & 31];
    float* out = col < C ? dw : db;
    if (out) out[col < C ? col : col - C] = r;
  }
}

// ----------------------------------------------------------------------------
// Rows wider than a CTA's registers: a CTA per row that reads it again for every sum (from L2), and a thread per
// column for dw and db.
// ----------------------------------------------------------------------------
__device__ __forceinline__ float cta_sum(float v, float* s) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
  for (int k = 0; k < LNB_MAX_WARPS; ++k) r += s[k];
  __syncthreads();
  return r;
}

template <typename T>
__global__ void __launch_bounds__(LNB_THREADS) layer_norm_wide_kernel(const __grid_constant__ LnFwdArgs a) {
  __shared__ float s[LNB_MAX_WARPS];
  grid_dep_wait();
  grid_dep_launch();
  const float inv_c = 1.0f / static_cast<float>(a.C);
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LNB_THREADS) v += to_float(x[c]);
    const float mean = cta_sum(v, s) * inv_c;
    v = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LNB_THREADS) v = fmaf(to_float(x[c]) - mean, to_float(x[c]) - mean, v);
    const float rstd = 1.0f / sqrtf(cta_sum(v, s) * inv_c + a.eps);
    T* out = static_cast<T*>(a.y) + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += LNB_THREADS)
      from_float(out + c, fmaf((to_float(x[c]) - mean) * rstd, a.w ? a.w[c] : 1.f, a.b ? a.b[c] : 0.f));
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(LNB_THREADS) layer_norm_backward_wide_kernel(const __grid_constant__ LnBwdArgs a) {
  __shared__ float s[LNB_MAX_WARPS];
  grid_dep_wait();
  grid_dep_launch();
  const float inv_c = 1.0f / static_cast<float>(a.C);
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgu = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LNB_THREADS) {
      const float g = to_float(dy[c]) * (a.w ? a.w[c] : 1.f);
      sg += g;
      sgu = fmaf(g, (to_float(x[c]) - mean) * rstd, sgu);
    }
    const float mg = cta_sum(sg, s) * inv_c, mgu = cta_sum(sgu, s) * inv_c;
    T* out = static_cast<T*>(a.dx) + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += LNB_THREADS) {
      const float u = (to_float(x[c]) - mean) * rstd;
      from_float(out + c, rstd * (fmaf(to_float(dy[c]), a.w ? a.w[c] : 1.f, -mg) - u * mgu));
    }
  }
}

// a CTA: 256 columns, rows blockIdx.y, + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_backward_wide_columns_kernel(const __grid_constant__ LnBwdArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.f, db = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float dy = to_float(static_cast<const T*>(a.dy)[row * a.lddy + c]);
    dw = fmaf(dy, (to_float(static_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row], dw);
    db += dy;
  }
  a.partial[(static_cast<long>(blockIdx.y) * 2) * a.C + c] = dw;
  a.partial[(static_cast<long>(blockIdx.y) * 2 + 1) * a.C + c] = db;
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
// How a width is cut up: a team of `warps` warps (or of `lanes` lanes of one) holds a row in nv pieces of vec values a
// thread.
struct LnShape {
  int vec, nv, lanes, warps, teams;
};

// As many pieces a thread as leave no more places idle than fewer would (a wide team spends more on its barrier), up to 16
// values of bf16 and 8 of fp32, whose two rows in flight take as many registers; 16 where nothing else holds the row.
LnShape ln_shape(int C, bool f32, bool aligned) {
  LnShape s;
  s.vec = aligned ? (f32 ? 4 : 8) : 1;
  const int nvec = C / s.vec;
  s.nv = 1;
  s.lanes = 32;
  s.warps = 1;
  if (nvec <= 32) {
    while (s.lanes > 4 && nvec <= s.lanes / 2) s.lanes /= 2;
  } else {
    long best = -1;
    for (int most = s.vec == 8 ? 16 : 8; best < 0 && most <= LNB_PER_THREAD; most *= 2)
      for (int nv = 1; nv * s.vec <= most; nv = s.vec == 1 && nv == 1 ? 4 : 2 * nv) {
        const int warps = (nvec + 32 * nv - 1) / (32 * nv);
        if (warps > LNB_MAX_WARPS) continue;
        const long places = static_cast<long>(warps) * nv;
        if (best < 0 || places <= best) { best = places; s.nv = nv; s.warps = warps; }
      }
  }
  s.teams = s.warps > 1 ? LNB_MAX_WARPS / s.warps : LNB_THREADS / s.lanes;
  return s;
}

bool row_aligned(const void* p, long ld, bool f32) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * (f32 ? 4 : 2)) % 16 == 0;
}

int cta_threads(const LnShape& s) { return s.teams * (s.warps > 1 ? 32 * s.warps : s.lanes); }

// CTAs for `rows`; few rows: no more teams in one than cover the SMs with a row each
int fit_teams(LnShape* s, long rows, int sms) {
  const long want = (rows + sms - 1) / sms;
  const int unit = s->warps > 1 ? 1 : 32 / s->lanes;  // teams of a whole warp
  if (want < s->teams) s->teams = static_cast<int>((want + unit - 1) / unit * unit);
  const long ctas = (rows + s->teams - 1) / s->teams;
  return static_cast<int>(ctas < sms ? ctas : sms);
}

// f.template run<T, VEC, NV, LANES>() of the shape
template <typename T, int VEC, typename F>
int with_pieces(const LnShape& s, const F& f) {
  if (s.lanes == 4) return f.template run<T, VEC, 1, 4>();
  if (s.lanes == 8) return f.template run<T, VEC, 1, 8>();
  if (s.lanes == 16) return f.template run<T, VEC, 1, 16>();
  if (s.nv == 1) return f.template run<T, VEC, 1, 32>();
  if constexpr (VEC > 1) {
    if (s.nv == 2) return f.template run<T, VEC, 2, 32>();
  }
  if constexpr (VEC == 1 || VEC == 4) {
    if (s.nv == 4) return f.template run<T, VEC, 4, 32>();
  }
  if constexpr (VEC == 1) {
    if (s.nv == 8) return f.template run<T, 1, 8, 32>();
    if (s.nv == 16) return f.template run<T, 1, 16, 32>();
  }
  set_last_error("layer_norm: no kernel for %d pieces", s.nv);
  return ST_UNSUPPORTED;
}
template <typename F>
int with_shape(const LnShape& s, bool f32, const F& f) {
  if (f32) return s.vec == 4 ? with_pieces<float, 4>(s, f) : with_pieces<float, 1>(s, f);
  return s.vec == 8 ? with_pieces<bf16, 8>(s, f) : with_pieces<bf16, 1>(s, f);
}

struct LaunchForward {
  const LnFwdArgs& a;
  int grid, threads;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, int LANES>
  int run() const {
    launch_dependent(layer_norm_kernel<T, VEC, NV, LANES>, grid, threads, 0, stream, a);
    return after_launch("layer_norm_kernel");
  }
};

struct LaunchBackward {
  const LnBwdArgs& a;
  int grid, threads;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, int LANES>
  int run() const {
    auto kern = layer_norm_backward_kernel<T, VEC, NV, LANES>;
    const size_t smem = 2 * sizeof(float) * a.C;
    if (smem > 48 * 1024 - 1024) {
      int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               2 * static_cast<int>(sizeof(float)) * LNB_MAX_C),
                          "cudaFuncSetAttribute(layer_norm_backward)");
      if (rc) return rc;
    }
    launch_dependent(kern, grid, threads, smem, stream, a);
    return after_launch("layer_norm_backward_kernel");
  }
};

// widest row that a CTA's registers hold
bool row_fits(int C, const LnShape& s) {
  return C <= s.vec * 32 * s.nv * s.warps;
}

constexpr int LNB_WIDE_PARTS = 64;  // row shares of the thread-per-column kernel

}  // namespace

int launch_layer_norm(const void* x, long ldx, int f32, const float* w, const float* b, float eps, void* y, float* mean,
                      float* rstd, long rows, int C, cudaStream_t stream) {
  LnFwdArgs a = {x, ldx, w, b, y, mean, rstd, rows, C, 1, 1, eps};
  const int sms = device_sm_count();
  LnShape s = ln_shape(C, f32 != 0, C % (f32 ? 4 : 8) == 0 && row_aligned(x, ldx, f32) && row_aligned(y, C, f32));
  if (!row_fits(C, s)) {
    const int grid = static_cast<int>(rows < 4L * sms ? rows : 4L * sms);
    launch_dependent(f32 ? layer_norm_wide_kernel<float> : layer_norm_wide_kernel<bf16>, grid, LNB_THREADS, 0, stream, a);
    return after_launch("layer_norm_wide_kernel");
  }
  const int grid = fit_teams(&s, rows, sms);
  a.warps = s.warps;
  a.teams = s.teams;
  return with_shape(s, f32 != 0, LaunchForward{a, grid, cta_threads(s), stream});
}

// room for the partial rows of dw and db: one per CTA
size_t layer_norm_backward_scratch_bytes(long rows, int C) {
  if (rows <= 0 || C <= 0) return 0;
  const int sms = device_sm_count();
  const long parts = sms > LNB_WIDE_PARTS ? sms : LNB_WIDE_PARTS;
  return static_cast<size_t>(rows < parts ? rows : parts) * 2 * C * sizeof(float);
}

int launch_layer_norm_backward(const void* dy, long lddy, const void* x, long ldx, int f32, const float* w,
                               const float* mean, const float* rstd, void* dx, float* dw, float* db, long rows, int C,
                               float* scratch, cudaStream_t stream) {
  LnBwdArgs a = {dy, lddy, x, ldx, w, mean, rstd, dx, scratch, rows, C, 1, 1};
  const int sms = device_sm_count();
  int parts = 0;
  if (rows > 0) {
    LnShape s = ln_shape(C, f32 != 0, C % (f32 ? 4 : 8) == 0 && row_aligned(x, ldx, f32) && row_aligned(dy, lddy, f32) &&
                                          row_aligned(dx, C, f32));
    if (!row_fits(C, s)) {
      // the columns first: dx may lie where x or dy does
      parts = static_cast<int>(rows < LNB_WIDE_PARTS ? rows : LNB_WIDE_PARTS);
      launch_dependent(f32 ? layer_norm_backward_wide_columns_kernel<float> : layer_norm_backward_wide_columns_kernel<bf16>,
                       dim3((C + 255) / 256, parts), 256, 0, stream, a);
      int rc = after_launch("layer_norm_backward_wide_columns_kernel");
      if (rc) return rc;
      const int grid = static_cast<int>(rows < 4L * sms ? rows : 4L * sms);
      launch_dependent(f32 ? layer_norm_backward_wide_kernel<float> : layer_norm_backward_wide_kernel<bf16>, grid,
                       LNB_THREADS, 0, stream, a);
      rc = after_launch("layer_norm_backward_wide_kernel");
      if (rc) return rc;
    } else {
      parts = fit_teams(&s, rows, sms);
      a.warps = s.warps;
      a.teams = s.teams;
      int rc = with_shape(s, f32 != 0, LaunchBackward{a, parts, cta_threads(s), stream});
      if (rc) return rc;
    }
  }
  launch_dependent(layer_norm_columns_kernel, (2 * C + 31) / 32, 256, 0, stream, scratch, parts, C, dw, db);
  return after_launch("layer_norm_columns_kernel");
}

}  // namespace sd3
