// Per-head RMS norm of the queries and keys of a packed q|k|v buffer, and the rotation of both by the events'
// positions, in one pass (forward, backward), and the same on the way into a paged key / value cache.
//
// One head of one token, x in R^hd, R = 2 * (number of frequencies) <= hd, angles a_i = pos * inv_freq_i:
//   z = w * x * r,  r = 1 / sqrt(mean(x^2) + eps)                    (no weights: z = x)
//   y_i = z_i cos a_i - z_{i+R/2} sin a_i,  y_{i+R/2} = z_{i+R/2} cos a_i + z_i sin a_i   (i < R/2),  y_j = z_j (j >= R)
// Backward, u = dy rotated by -a: dw = sum over tokens and heads of u * x r,  g = u * w,
//   dx = r * (g - x * r^2 * mean(g * x)).
//
// The angle is the exact product of two f32 (or of an integer below 2^29 and an f32) in f64, reduced to turns in f64:
// event times reach 1e5..1e6 minutes, where an f32 product is off by up to 0.03 rad. The reduced turn in [-1/2, 1/2]
// goes to f32 (off by at most 2^-26 turns) and through sincospi.
//
// All three are bound by HBM: the packed row is read and written once. A lane owns V elements of a head and their V
// rotation partners (two 16-B accesses each way, so the rotation needs no exchange between lanes), the head's lanes
// are neighbours in one wave (the norm's sum is a short DPP butterfly), and a thread keeps its (head, chunk) while it
// walks tokens, so that weights stay in registers and the backward sums dw there. The sines and cosines of a token
// are shared by its 2 H heads: the workgroup computes those of a run of tokens once, into LDS.
#include "common.h"

#include <algorithm>

using namespace esgpt;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxD = 16384;  // H * hd: keeps the kernels' 32-bit divisions exact (fdiv)

enum : int { MODE_FWD = 0, MODE_BWD = 1, MODE_APPEND = 2 };
constexpr int64_t kMasked = -1, kNowhere = -2;  // append: a padded row; a row without a place in the cache

struct RopeArgs {
  const void* x;         // raw packed rows [N, 3D]
  const void* dy;        // backward: the outputs' gradient [N, 3D]
  void* out;             // forward: [N, 3D]; backward: dx [N, 3D]; append: q [N, D]
  const float* w[2];     // q, k norm weights [hd] (both or none)
  const void* pos;       // [N] f32 or int64
  const float* inv_freq; // [R2]
  float* part;           // backward: [gridDim.x, 2, hd] partial sums of dw
  int64_t N;
  int pos_i64, R2, H, hd, C, GP, slots, passes, run;
  float eps;
  uint64_t magic_r, magic_v;  // division by R2 and by a token's 16-B chunks of v
  // append
  const uint8_t* row_mask;    // [S, Lq] or null
  const int32_t* past;        // [S]
  const int32_t* page_table;  // [S, table_w]
  void* k_pages;              // [n_pages, H, ps, hd]
  void* v_pages;
  int32_t* err;
  int64_t n_pages, table_w;
  int Lq, ps;
};

__device__ __forceinline__ void turn_sincos(const RopeArgs& a, int64_t n, int i, float& s, float& c) {
  const double p = a.pos_i64 ? (double)reinterpret_cast<const int64_t*>(a.pos)[n]
                             : (double)reinterpret_cast<const float*>(a.pos)[n];
  const double t = p * (double)a.inv_freq[i] * 0.15915494309189533577;  // turns
  sincospif(2.f * (float)(t - rint(t)), &s, &c);
}

// Sum over the GP (power of two) neighbouring lanes of one head; every lane ends with the sum.
__device__ __forceinline__ float group_sum(float v, int gp) {
  if (gp > 1) v += dpp_mov<0xB1>(v);
  if (gp > 2) v += dpp_mov<0x4E>(v);
  if (gp > 4) v += dpp_mov<0x141>(v);
  if (gp > 8) v += dpp_mov<0x140>(v);
  if (gp > 16) {
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  if (gp > 32) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Chunk {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> ld(const T* p) { return *reinterpret_cast<const Chunk<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void st(T* p, const float (&v)[V]) {
  Chunk<T, V> c;
#pragma unroll
  for (int j = 0; j < V; ++j) c.e[j] = from_f32<T>(v[j]);
  *reinterpret_cast<Chunk<T, V>*>(p) = c;
}

// Rows [0, i) of a sequence's mask that are set, by the whole workgroup (append: where the first token of the run
// lands). `red`: one int per wave.
__device__ __forceinline__ int mask_prefix(const uint8_t* m, int i, int* red) {
  int c = 0;
  for (int j = threadIdx.x; j < i; j += blockDim.x) c += m[j] != 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane_id() == 0) red[threadIdx.x >> 6] = c;
  __syncthreads();
  int t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += red[w];
  return t;
}

// q = n / d for n, d < 2^16 by the host's magic = ceil(2^32 / d).
__device__ __forceinline__ int fdiv(int n, uint64_t magic) { return (int)(((uint64_t)(uint32_t)n * magic) >> 32); }

// blockDim.x = the slots * 2H * GP lanes of `slots` tokens, rounded up to whole waves (passes > 1: one token's
// 2H * GP lanes in passes of 256). Run r of the grid-strided list of runs covers tokens [r * run, (r + 1) * run).
template <typename T, int V, int MODE, bool NORM>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
  extern __shared__ __align__(16) char smem[];
  const int H = a.H, hd = a.hd, R2 = a.R2, D = H * hd, GP = a.GP;
  const int64_t ld_x = 3 * (int64_t)D;
  const int ipt = 2 * H * GP;  // lanes of one token
  float2* cs = reinterpret_cast<float2*>(smem);                                            // [run][R2]
  int64_t* dst = reinterpret_cast<int64_t*>(smem + (size_t)a.run * R2 * sizeof(float2));   // append: [run]
  const int tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  T* out = reinterpret_cast<T*>(a.out);
  const int64_t n_runs = (a.N + a.run - 1) / a.run;
  const float inv_hd = 1.f / (float)hd;

  for (int pass = 0; pass < a.passes; ++pass) {
    const int item = a.passes > 1 ? pass * kThreads + tid : tid % ipt;
    const int slot = a.passes > 1 ? 0 : tid / ipt;
    const int hh = item / GP, c = item & (GP - 1);  // hh < H: query head hh, else key head hh - H
    const bool live = slot < a.slots && hh < 2 * H;
    const bool on = live && c < a.C;  // a group's lanes past C carry zeros through its sums
    const int isk = hh >= H;
    const int e = on ? c * V : 0;
    const bool rot = e < R2;
    const int lo = rot ? e : e + R2;  // the chunk and its partner in the head
    const int hi = lo + (rot ? R2 : hd / 2 - R2);
    const int64_t col = (int64_t)hh * hd;  // q heads, then k heads: contiguous in the packed row
    float wl[V], wh[V], al[V], ah[V];      // weights; sums of dw
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wl[j] = on ? a.w[isk][lo + j] : 0.f;
        wh[j] = on ? a.w[isk][hi + j] : 0.f;
        al[j] = ah[j] = 0.f;
      }
    }
    for (int64_t r = blockIdx.x; r < n_runs; r += gridDim.x) {
      const int64_t n0 = r * a.run;
      const int nt = (int)min((int64_t)a.run, a.N - n0);
      __syncthreads();  // the previous run's readers of cs / dst
      for (int i = tid; i < nt * R2; i += blockDim.x) {
        const int t = fdiv(i, a.magic_r);
        float sn, cn;
        turn_sincos(a, n0 + t, i - t * R2, sn, cn);
        cs[i] = make_float2(cn, sn);
      }
      if constexpr (MODE == MODE_APPEND) {
        int* red = reinterpret_cast<int*>(dst + a.run);
        const int64_t s0 = n0 / a.Lq;
        const int before = a.row_mask ? mask_prefix(a.row_mask + s0 * a.Lq, (int)(n0 - s0 * a.Lq), red) : 0;
        for (int t = tid; t < nt; t += blockDim.x) {
          const int64_t n = n0 + t, s = n / a.Lq;
          int64_t d = kMasked;
          if (!a.row_mask || a.row_mask[n]) {
            int64_t row = n - s * a.Lq;
            if (a.row_mask) {
              row = s == s0 ? before : 0;
              for (int64_t j = max(n0, s * a.Lq); j < n; ++j) row += a.row_mask[j] != 0;
            }
            const int64_t past = a.past[s];
            row += past;
            d = kNowhere;
            if (past >= 0 && row < a.table_w * a.ps) {
              const int64_t page = a.page_table[s * a.table_w + row / a.ps];
              if (page >= 0 && page < a.n_pages) d = (page * H * a.ps + row % a.ps) * hd;
            }
            if (d == kNowhere && pass == 0) set_err(a.err, ESGPT_FLAG_BAD_PAGE);
          }
          dst[t] = d;
        }
      }
      __syncthreads();

      if (live) {
        for (int t = slot; t < nt; t += a.slots) {
          const int64_t n = n0 + t;
          float fl[V], fh[V];
          if (on) {
            const T* xp = x + n * ld_x + col;
            const Chunk<T, V> xl = ld<T, V>(xp + lo), xh = ld<T, V>(xp + hi);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              fl[j] = to_f32(xl.e[j]);
              fh[j] = to_f32(xh.e[j]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) fl[j] = fh[j] = 0.f;
          }
          float cn[V], sn[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 v = rot && R2 > 0 ? cs[t * R2 + e + j] : make_float2(1.f, 0.f);
            cn[j] = v.x;
            sn[j] = v.y;
          }
          float rstd = 1.f;
          if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) ss = fmaf(fl[j], fl[j], fmaf(fh[j], fh[j], ss));
            rstd = rsqrtf(fmaf(group_sum(ss, GP), inv_hd, a.eps));
          }
          float yl[V], yh[V];
          if constexpr (MODE == MODE_BWD) {
            float gl[V], gh[V];
            if (on) {
              const T* dp = dy + n * ld_x + col;
              const Chunk<T, V> dl = ld<T, V>(dp + lo), dh = ld<T, V>(dp + hi);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const float p = to_f32(dl.e[j]), q = to_f32(dh.e[j]);
                gl[j] = rot ? fmaf(p, cn[j], q * sn[j]) : p;
                gh[j] = rot ? fmaf(q, cn[j], -p * sn[j]) : q;
              }
            } else {
#pragma unroll
              for (int j = 0; j < V; ++j) gl[j] = gh[j] = 0.f;
            }
            if constexpr (NORM) {
              float gx = 0.f;
#pragma unroll
              for (int j = 0; j < V; ++j) {
                al[j] = fmaf(gl[j], fl[j] * rstd, al[j]);
                ah[j] = fmaf(gh[j], fh[j] * rstd, ah[j]);
                gl[j] *= wl[j];
                gh[j] *= wh[j];
                gx = fmaf(gl[j], fl[j], fmaf(gh[j], fh[j], gx));
              }
              const float m = group_sum(gx, GP) * inv_hd * rstd * rstd;
#pragma unroll
              for (int j = 0; j < V; ++j) {
                gl[j] = rstd * (gl[j] - fl[j] * m);
                gh[j] = rstd * (gh[j] - fh[j] * m);
              }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
              yl[j] = gl[j];
              yh[j] = gh[j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float p = NORM ? fl[j] * rstd * wl[j] : fl[j], q = NORM ? fh[j] * rstd * wh[j] : fh[j];
              yl[j] = rot ? fmaf(p, cn[j], -q * sn[j]) : p;
              yh[j] = rot ? fmaf(q, cn[j], p * sn[j]) : q;
            }
          }
          if (!on) continue;
          T* op = out + n * ld_x + col;
          if constexpr (MODE == MODE_APPEND) {
            const int64_t d = dst[t];
            if (!isk) {
              op = out + n * D + col;
              if (d == kMasked) {
#pragma unroll
                for (int j = 0; j < V; ++j) yl[j] = yh[j] = 0.f;
              }
            } else {
              if (d < 0) continue;
              op = reinterpret_cast<T*>(a.k_pages) + d + (int64_t)(hh - H) * a.ps * hd;
            }
          }
          st<T, V>(op + lo, yl);
          st<T, V>(op + hi, yh);
        }
      }
      if (pass == 0) {  // v: copied, 16 B a lane
        constexpr int E = 16 / (int)sizeof(T);
        const int vch = D / E;
        const T* vp = (MODE == MODE_BWD ? dy : x) + 2 * D;
        for (int i = tid; i < nt * vch; i += blockDim.x) {
          const int t = fdiv(i, a.magic_v), f = (i - t * vch) * E;
          const uint4 v = *reinterpret_cast<const uint4*>(vp + (n0 + t) * ld_x + f);
          if constexpr (MODE == MODE_APPEND) {
            const int64_t d = dst[t];
            if (d < 0) continue;
            const int h = f / hd;
            *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.v_pages) + d + (int64_t)h * a.ps * hd + (f - h * hd)) = v;
          } else {
            *reinterpret_cast<uint4*>(out + (n0 + t) * ld_x + 2 * D + f) = v;
          }
        }
      }
    }

    if constexpr (MODE == MODE_BWD && NORM) {
      // dw of this workgroup: the lanes that hold one element (its chunk in every token slot and head), summed in a
      // fixed order
      float* buf = reinterpret_cast<float*>(smem);  // [lanes][2V]
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        buf[tid * 2 * V + j] = al[j];
        buf[tid * 2 * V + V + j] = ah[j];
      }
      __syncthreads();
      for (int o = tid; o < 2 * hd; o += blockDim.x) {
        const int k = o >= hd, el = o - k * hd, tail = hd / 2 - R2;
        int half, ee;  // element el is element ee of the head's chunks, in the lower or the upper half
        if (el < 2 * R2) {
          half = el >= R2;
          ee = el - half * R2;
        } else {
          half = el - 2 * R2 >= tail;
          ee = el - R2 - half * tail;
        }
        const int off = half * V + ee % V, cc = ee / V;
        float sum = 0.f;
        if (a.passes > 1) {
          const int per = kThreads / GP;
          for (int g = 0; g < per; ++g) {
            const int hg = pass * per + g;
            if (hg < 2 * H && (hg >= H) == (k != 0)) sum += buf[(g * GP + cc) * 2 * V + off];
          }
        } else {
          for (int s = 0; s < a.slots; ++s)
            for (int h = 0; h < H; ++h) sum += buf[(s * ipt + (k * H + h) * GP + cc) * 2 * V + off];
        }
        float* p = a.part + (int64_t)blockIdx.x * 2 * hd + o;
        *p = pass > 0 ? *p + sum : sum;  // the same thread every pass
      }
    }
  }
}

struct Plan {
  int V, C, GP, slots, passes, block, run;
  int64_t grid;
  size_t lds;
};

// V: the widest access (up to 16 B) that the rotated half and half of what is not rotated are whole multiples of.
// The workgroup takes as many tokens at once as give it up to 256 lanes, and one to four such sets per run: more
// tokens per run cost fewer barriers and workgroups, while fewer keep the chip full (kRuns runs at least).
Plan make_plan(int64_t N, int64_t H, int64_t hd, int64_t R, int dtype, int mode) {
  Plan p;
  const int64_t R2 = R / 2, tail = hd / 2 - R2;
  int V = dtype == ESGPT_BF16 ? 8 : 4;
  while (R2 % V || tail % V) V /= 2;
  p.V = V;
  p.C = (int)(hd / 2 / V);
  p.GP = 1;
  while (p.GP < p.C) p.GP *= 2;
  const int64_t ipt = 2 * H * p.GP;
  p.passes = (int)cdiv(ipt, kThreads);
  p.slots = p.passes > 1 ? 1 : (int)(kThreads / ipt);
  p.block = p.passes > 1 ? kThreads : (int)(cdiv(p.slots * ipt, 64) * 64);
  const int64_t kRuns = mode == MODE_BWD ? 1024 : 2048;
  const int64_t sets = std::max<int64_t>(1, std::min<int64_t>(4, N / (p.slots * kRuns)));
  p.run = (int)(p.slots * sets);
  p.grid = std::min<int64_t>(cdiv(N, p.run), mode == MODE_BWD ? 1024 : (int64_t)1 << 20);
  p.lds = (size_t)p.run * R2 * sizeof(float2);
  if (mode == MODE_APPEND) p.lds += (size_t)p.run * 8 + 4 * 4;
  if (mode == MODE_BWD) p.lds = std::max(p.lds, (size_t)p.block * 2 * V * sizeof(float));
  return p;
}

template <typename T, int MODE, bool NORM>
void launch_v(const Plan& p, const RopeArgs& a, hipStream_t st) {
  const dim3 g((unsigned)p.grid), b(p.block);
  constexpr int VM = 16 / (int)sizeof(T);
  if (p.V == VM) rope_kernel<T, VM, MODE, NORM><<<g, b, p.lds, st>>>(a);
  else if (p.V == VM / 2) rope_kernel<T, VM / 2, MODE, NORM><<<g, b, p.lds, st>>>(a);
  else if (p.V == 1) rope_kernel<T, 1, MODE, NORM><<<g, b, p.lds, st>>>(a);
  else if constexpr (VM == 8) rope_kernel<T, 2, MODE, NORM><<<g, b, p.lds, st>>>(a);
}

template <int MODE>
void launch(const Plan& p, const RopeArgs& a, int dtype, hipStream_t st) {
  if (dtype == ESGPT_BF16) {
    if (a.w[0]) launch_v<bf16, MODE, true>(p, a, st);
    else launch_v<bf16, MODE, false>(p, a, st);
  } else {
    if (a.w[0]) launch_v<float, MODE, true>(p, a, st);
    else launch_v<float, MODE, false>(p, a, st);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The arguments that all three share; false: one of them does not fit.
bool rope_ok(const void* x, const float* q_w, const float* k_w, const void* pos, int pos_dtype, const float* inv_freq,
             int64_t R, int64_t N, int64_t H, int64_t hd, float eps, int dtype) {
  return N >= 0 && H > 0 && hd > 0 && hd <= 128 && H <= kMaxD / hd && hd % (dtype == ESGPT_BF16 ? 8 : 4) == 0 &&
         (dtype == ESGPT_F32 || dtype == ESGPT_BF16) && R >= 0 && R % 2 == 0 && R <= hd &&
         (R == 0 || N == 0 || (pos && inv_freq)) && (pos_dtype == ESGPT_POS_F32 || pos_dtype == ESGPT_POS_I64) &&
         (q_w != nullptr) == (k_w != nullptr) && eps >= 0.f && (N == 0 || (x && aligned16(x)));
}

RopeArgs rope_args(const Plan& p, const void* x, const float* q_w, const float* k_w, const void* pos, int pos_dtype,
                   const float* inv_freq, int64_t R, int64_t N, int64_t H, int64_t hd, float eps, int dtype) {
  RopeArgs a{};
  a.x = x;
  a.w[0] = q_w;
  a.w[1] = k_w;
  a.pos = pos;
  a.pos_i64 = pos_dtype == ESGPT_POS_I64;
  a.inv_freq = inv_freq;
  a.N = N;
  a.R2 = (int)(R / 2);
  a.H = (int)H;
  a.hd = (int)hd;
  a.C = p.C;
  a.GP = p.GP;
  a.slots = p.slots;
  a.passes = p.passes;
  a.run = p.run;
  a.eps = eps;
  const uint64_t vch = (uint64_t)(H * hd) / (dtype == ESGPT_BF16 ? 8 : 4);
  a.magic_r = R ? ((1ull << 32) + R / 2 - 1) / (R / 2) : 0;
  a.magic_v = ((1ull << 32) + vch - 1) / vch;
  return a;
}

}  // namespace

extern "C" {

int esgpt_qk_norm_rope_fwd(const void* qkv, const float* q_w, const float* k_w, const void* pos, int pos_dtype,
                           const float* inv_freq, int64_t R, int64_t N, int64_t H, int64_t hd, float eps, void* out,
                           int dtype, void* stream) {
  ESGPT_REQUIRE(rope_ok(qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, N, H, hd, eps, dtype));
  if (N == 0) return ESGPT_OK;
  ESGPT_REQUIRE(out && aligned16(out));
  const Plan p = make_plan(N, H, hd, R, dtype, MODE_FWD);
  RopeArgs a = rope_args(p, qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, N, H, hd, eps, dtype);
  a.out = out;
  launch<MODE_FWD>(p, a, dtype, as_stream(stream));
  ESGPT_LAUNCH_CHECK();
  return ESGPT_OK;
}

size_t esgpt_qk_norm_rope_bwd_workspace(int64_t N, int64_t H, int64_t hd, int64_t R, int dtype) {
  if (N <= 0 || H <= 0 || hd <= 0 || hd > 128 || R < 0 || R > hd) return 0;
  return (size_t)make_plan(N, H, hd, R, dtype, MODE_BWD).grid * 2 * hd * sizeof(float);
}

int esgpt_qk_norm_rope_bwd(const void* dout, const void* qkv, const float* q_w, const float* k_w, const void* pos,
                           int pos_dtype, const float* inv_freq, int64_t R, int64_t N, int64_t H, int64_t hd,
                           float eps, void* dqkv, float* dw, void* workspace, size_t workspace_bytes, int dtype,
                           void* stream) {
  ESGPT_REQUIRE(rope_ok(qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, N, H, hd, eps, dtype));
  ESGPT_REQUIRE(!q_w || (dw && aligned16(dw)));
  hipStream_t st = as_stream(stream);
  if (N == 0) {
    if (q_w && zero_async(dw, 2 * hd * sizeof(float), st) != hipSuccess) return ESGPT_ERR_LAUNCH;
    return ESGPT_OK;
  }
  ESGPT_REQUIRE(dout && dqkv && aligned16(dout) && aligned16(dqkv));
  const Plan p = make_plan(N, H, hd, R, dtype, MODE_BWD);
  RopeArgs a = rope_args(p, qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, N, H, hd, eps, dtype);
  a.dy = dout;
  a.out = dqkv;
  if (q_w) {
    ESGPT_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= p.grid * 2 * hd * sizeof(float));
    a.part = reinterpret_cast<float*>(workspace);
  }
  launch<MODE_BWD>(p, a, dtype, st);
  ESGPT_LAUNCH_CHECK();
  if (!q_w) return ESGPT_OK;
  const esgpt_colsum_job job{a.part, p.grid, 2 * hd, dw};
  return esgpt_colsum_jobs(&job, 1, stream);
}

int esgpt_kv_append_paged(const void* qkv, const float* q_w, const float* k_w, const void* pos, int pos_dtype,
                          const float* inv_freq, int64_t R, float eps, const uint8_t* row_mask, const int32_t* past,
                          const int32_t* page_table, int64_t table_w, void* k_pages, void* v_pages, int64_t n_pages,
                          int64_t page_size, void* q, int64_t S, int64_t Lq, int64_t H, int64_t hd, int dtype,
                          int32_t* err, void* stream) {
  ESGPT_REQUIRE(S >= 0 && Lq >= 0 && Lq < (int64_t)1 << 31 && S < (int64_t)1 << 31);
  ESGPT_REQUIRE(rope_ok(qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, S * Lq, H, hd, eps, dtype));
  ESGPT_REQUIRE(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0 && table_w >= 0 &&
                n_pages >= 0);
  if (S * Lq == 0) return ESGPT_OK;
  ESGPT_REQUIRE(past && q && aligned16(q) && (table_w == 0 || page_table) &&
                (n_pages == 0 || (k_pages && v_pages && aligned16(k_pages) && aligned16(v_pages))));
  const Plan p = make_plan(S * Lq, H, hd, R, dtype, MODE_APPEND);
  RopeArgs a = rope_args(p, qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, S * Lq, H, hd, eps, dtype);
  a.out = q;
  a.row_mask = row_mask;
  a.past = past;
  a.page_table = page_table;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.err = err;
  a.n_pages = n_pages;
  a.table_w = table_w;
  a.Lq = (int)Lq;
  a.ps = (int)page_size;
  launch<MODE_APPEND>(p, a, dtype, as_stream(stream));
  ESGPT_LAUNCH_CHECK();
  return ESGPT_OK;
}

}  // extern "C"
