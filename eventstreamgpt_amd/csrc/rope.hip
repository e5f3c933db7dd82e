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
// are shared by its 2 H heads: the workgroup computes those of a run of tokens once, into LDS, while the loads of its
// first tokens are in flight; the next token's loads follow the current one's last use of the registers.
// Measured (hd 64, bf16): 65,536 tokens of 8 heads forward 71 us (5.7 TB/s), backward 112 us + 5 of dw sum (4.8 TB/s; four
// waves per SIMD, at three it was 167), a large copy's rate on this card being 4.95; 32 x 1024 rows appended, a third of
// them padding, 4 heads 19 us (3.8 TB/s); 512 sequences' single rows 6.0 us, the chain of past, page id and store.
#include "common.h"

#include <algorithm>

using namespace esgpt;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRun = 512;      // tokens of a run
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
  uint64_t magic_r;  // division by R2
  // append
  const uint8_t* row_mask;    // [S, Lq] or null
  const int32_t* past;        // [S]
  const int32_t* page_table;  // [S, table_w]
  void* k_pages;              // [n_pages, H, ps, hd]
  void* v_pages;
  int32_t* err;
  int64_t n_pages, table_w;
  int Lq, ps, psl;  // psl: log2 of the page size
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

// Rows [0, i) of a sequence's mask that are set, counted by this wave's share; the waves' counts go to red.
__device__ __forceinline__ void mask_count(const uint8_t* m, int i, int* red) {
  int c = 0;
#pragma unroll 4
  for (int j = threadIdx.x; j < i; j += blockDim.x) c += m[j] != 0;
  const float sum = wave_sum((float)c);  // below 2^24: exact
  if (lane_id() == 0) red[threadIdx.x >> 6] = (int)sum;
}

// q = n / d for n, d < 2^16 by the host's magic = ceil(2^32 / d).
__device__ __forceinline__ int fdiv(int n, uint64_t magic) { return (int)(((uint64_t)(uint32_t)n * magic) >> 32); }

// Append: the element offset (head 0) of the cache row of each of the run's nt <= 64 tokens, one lane of the first wave
// each; kMasked or kNowhere. A token's row counts the kept rows of its sequence before it: those before the run from
// `red`, those in the run from the wave's ballot. What does not depend on the count is loaded before it (Token).
struct Token {
  int s, i;  // sequence, row of it
  bool keep;
  int past;
};
__device__ __forceinline__ Token token_of(const RopeArgs& a, int n, bool in) {
  Token k{n / a.Lq, 0, in, 0};
  k.i = n - k.s * a.Lq;
  if (!in) return k;
  k.past = a.past[k.s];
  if (a.row_mask) k.keep = a.row_mask[n] != 0;
  return k;
}
__device__ __forceinline__ int64_t place(const RopeArgs& a, const Token& k, const int* red, bool report) {
  const int lane = lane_id();
  int64_t row = k.i;
  if (a.row_mask) {
    uint64_t before = __ballot(k.keep) & (lane ? ~0ull >> (64 - lane) : 0ull);
    if (lane > k.i) before &= ~0ull << (lane - k.i);  // the sequence began within the run: its own tokens only
    row = __popcll(before);
    if (lane <= k.i)
      for (int w = 0; w < (int)(blockDim.x >> 6); ++w) row += red[w];
  }
  if (!k.keep) return kMasked;
  row += k.past;
  if (k.past >= 0 && row < a.table_w << a.psl) {
    const int page = a.page_table[k.s * a.table_w + (row >> a.psl)];
    if (page >= 0 && page < a.n_pages) return (((int64_t)page * a.H << a.psl) + (row & (a.ps - 1))) * a.hd;
  }
  if (report) set_err(a.err, ESGPT_FLAG_BAD_PAGE);
  return kNowhere;
}

// blockDim.x = the slots * 2H * GP lanes of `slots` tokens, rounded up to whole waves (passes > 1: one token's
// 2H * GP lanes in passes of 256). Run r of the grid-strided list of runs covers tokens [r * run, (r + 1) * run).
template <typename T, int V, int MODE, bool NORM>
__global__ __launch_bounds__(kThreads, MODE == MODE_BWD ? 4 : 1) void rope_kernel(RopeArgs a) {
  extern __shared__ __align__(16) char smem[];
  const int H = a.H, hd = a.hd, R2 = a.R2, D = H * hd, GP = a.GP;
  const int64_t ld_x = 3 * (int64_t)D;
  const int ipt = 2 * H * GP;  // lanes of one token
  float* ws = reinterpret_cast<float*>(smem);                  // norm weights [2][hd]: in LDS, for the registers' sake
  float2* cs = reinterpret_cast<float2*>(ws + 2 * hd);         // [run][R2], 8 entries at least
  int64_t* dst = reinterpret_cast<int64_t*>(cs + max(a.run * R2, 8));  // append: [run]
  const int tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  T* out = reinterpret_cast<T*>(a.out);
  const int64_t n_runs = (a.N + a.run - 1) / a.run;
  const float inv_hd = 1.f / (float)hd;
  // Loads run a token ahead, but for the backward with norms: its registers are full (chunks of eight spill; chunks of four
  // gain 2 % or lose it). The backward without, 32,768 tokens of 8 heads bf16 48.6 -> 39.0 us.
  constexpr bool kAhead = !(MODE == MODE_BWD && NORM);

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
    const int64_t col = live ? (int64_t)hh * hd : 0;  // q heads, then k heads: contiguous in the packed row
    float al[V], ah[V];  // sums of dw
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < V; ++j) al[j] = ah[j] = 0.f;
      for (int i = tid; i < 2 * hd; i += blockDim.x) ws[i] = a.w[i >= hd][i >= hd ? i - hd : i];
    }
    const float* wt = ws + (live ? isk * hd : 0);
    // v is copied 16 B a lane: a token's vch chunks are at most its lanes, and neighbours in both
    constexpr int E = 16 / (int)sizeof(T);
    const int vch = D / E;
    const bool von = slot < a.slots && item < vch;
    const int vh = item * E / hd;  // append: the chunk's head

    for (int64_t r = blockIdx.x; r < n_runs; r += gridDim.x) {
      const int64_t n0 = r * a.run;
      const int nt = (int)min((int64_t)a.run, a.N - n0);
      Chunk<T, V> xl, xh, dl, dh;
      uint4 vv;
      // One token's loads, the same for every lane: one without a chunk of its own loads its group's first (or the
      // token's first) and stores nothing.
      auto fetch = [&](int64_t n) {
        const T* xp = x + n * ld_x + col;
        xl = ld<T, V>(xp + lo);
        xh = ld<T, V>(xp + hi);
        if constexpr (MODE == MODE_BWD) {
          const T* dp = dy + n * ld_x + col;
          dl = ld<T, V>(dp + lo);
          dh = ld<T, V>(dp + hi);
        }
        if constexpr (MODE != MODE_BWD) vv = *reinterpret_cast<const uint4*>(x + n * ld_x + 2 * D + (von ? item * E : 0));
      };
      // the first token's loads are in flight while the run's sines and cosines (and cache rows) are worked out
      Token tok;
      if constexpr (MODE == MODE_APPEND) tok = token_of(a, (int)n0 + min(tid, nt - 1), tid < nt);
      const int64_t n1 = min(n0 + slot, a.N - 1);
      bool keep = kAhead;
      if constexpr (MODE == MODE_APPEND) keep = !a.row_mask || a.row_mask[n1] != 0;
      if (keep) fetch(n1);
      __syncthreads();  // the previous run's readers of cs / dst
      for (int i = tid; i < nt * R2; i += blockDim.x) {
        const int t = fdiv(i, a.magic_r);
        float sn, cn;
        turn_sincos(a, n0 + t, i - t * R2, sn, cn);
        cs[i] = make_float2(cn, sn);
      }
      if constexpr (MODE == MODE_APPEND) {
        int* red = reinterpret_cast<int*>(dst + a.run);
        if (a.row_mask) {
          const int i0 = (int)n0 % a.Lq;
          mask_count(a.row_mask + n0 - i0, i0, red);
          __syncthreads();
        }
        if (tid < 64) {
          const int64_t d = place(a, tok, red, pass == 0);
          if (tid < nt) dst[tid] = d;
        }
      }
      __syncthreads();

      // the next token's loads, once this one's registers are free
      auto ahead = [&](int t) {
        const int u = t + a.slots;
        if (u >= nt) return;
        if (MODE == MODE_APPEND && dst[u] == kMasked) return;
        fetch(n0 + u);
      };
      for (int t = slot; t < nt; t += a.slots) {
        const int64_t n = n0 + t;
        int64_t d = 0;
        if constexpr (MODE == MODE_APPEND) {
          d = dst[t];
          if (d == kMasked) {  // padding: nothing is read, the query is zero
            if (on && !isk) {
              const float z[V] = {};
              st<T, V>(out + n * D + col + lo, z);
              st<T, V>(out + n * D + col + hi, z);
            }
            ahead(t);
            continue;
          }
        }
        if (!kAhead) fetch(n);
        if (von) {
          if constexpr (MODE == MODE_APPEND) {
            if (d >= 0)
              *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.v_pages) + d + (int64_t)vh * a.ps * hd + (item * E - vh * hd)) = vv;
          } else if constexpr (MODE == MODE_FWD) {
            *reinterpret_cast<uint4*>(out + n * ld_x + 2 * D + item * E) = vv;
          }
        }
        if (live) {
          const float2* ct = cs + (rot ? t * R2 + e : 0);  // V entries are there for any lane, used where rot
          float fl[V], fh[V], yl[V], yh[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            fl[j] = on ? to_f32(xl.e[j]) : 0.f;
            fh[j] = on ? to_f32(xh.e[j]) : 0.f;
          }
          if (MODE != MODE_BWD) ahead(t);
          float rstd = 1.f;
          if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) ss = fmaf(fl[j], fl[j], fmaf(fh[j], fh[j], ss));
            rstd = rsqrtf(fmaf(group_sum(ss, GP), inv_hd, a.eps));
          }
          if constexpr (MODE == MODE_BWD) {
            float gx = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              // a few LDS reads at a time: all of them at once do not fit 128 registers
              if (V == 8 && j % 2 == 0) __builtin_amdgcn_sched_barrier(0);
              const float p = on ? to_f32(dl.e[j]) : 0.f, q = on ? to_f32(dh.e[j]) : 0.f;
              const float2 v = ct[j];
              yl[j] = rot ? fmaf(p, v.x, q * v.y) : p;
              yh[j] = rot ? fmaf(q, v.x, -p * v.y) : q;
              if constexpr (NORM) {
                al[j] = fmaf(yl[j], fl[j] * rstd, al[j]);
                ah[j] = fmaf(yh[j], fh[j] * rstd, ah[j]);
                yl[j] *= wt[lo + j];
                yh[j] *= wt[hi + j];
                gx = fmaf(yl[j], fl[j], fmaf(yh[j], fh[j], gx));
              }
            }
            if (kAhead) ahead(t);
            if constexpr (NORM) {
              const float m = group_sum(gx, GP) * inv_hd * rstd * rstd;
#pragma unroll
              for (int j = 0; j < V; ++j) {
                yl[j] = rstd * (yl[j] - fl[j] * m);
                yh[j] = rstd * (yh[j] - fh[j] * m);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float p = NORM ? fl[j] * rstd * wt[lo + j] : fl[j], q = NORM ? fh[j] * rstd * wt[hi + j] : fh[j];
              const float2 v = ct[j];
              yl[j] = rot ? fmaf(p, v.x, -q * v.y) : p;
              yh[j] = rot ? fmaf(q, v.x, p * v.y) : q;
            }
          }
          bool store = on;
          T* op = out + n * ld_x + col;
          if constexpr (MODE == MODE_APPEND) {
            if (!isk) {
              op = out + n * D + col;
            } else {
              store = store && d >= 0;
              op = reinterpret_cast<T*>(a.k_pages) + d + (int64_t)(hh - H) * a.ps * hd;
            }
          }
          if (store) {
            st<T, V>(op + lo, yl);
            st<T, V>(op + hi, yh);
          }
        }
        if constexpr (MODE == MODE_BWD) {  // not among the token's first loads: no registers left to hold it
          if (von)
            *reinterpret_cast<uint4*>(out + n * ld_x + 2 * D + item * E) =
                *reinterpret_cast<const uint4*>(dy + n * ld_x + 2 * D + item * E);
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
      __syncthreads();  // the next pass writes the weights over buf
    }
  }
}

// dw = the workgroups' partial sums, in a fixed order: 16 columns a workgroup, 64 interleaved groups of rows.
__global__ __launch_bounds__(256) void dw_sum_kernel(const float* part, int64_t n, int width, float* dw) {
  __shared__ float4 s[64][4];
  const int c4 = threadIdx.x & 3, grp = threadIdx.x >> 2, col = blockIdx.x * 16 + 4 * c4;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < width) {
#pragma unroll 8
    for (int64_t r = grp; r < n; r += 64) {
      const float4 v = *reinterpret_cast<const float4*>(part + r * width + col);
      t.x += v.x;
      t.y += v.y;
      t.z += v.z;
      t.w += v.w;
    }
  }
  s[grp][c4] = t;
  for (int h = 32; h > 0; h >>= 1) {
    __syncthreads();
    if (grp < h) {
      const float4 v = s[grp + h][c4];
      t.x += v.x;
      t.y += v.y;
      t.z += v.z;
      t.w += v.w;
      s[grp][c4] = t;
    }
  }
  if (grp == 0 && col < width) *reinterpret_cast<float4*>(dw + col) = t;
}

struct Plan {
  int V, C, GP, slots, passes, block, run;
  int64_t grid;
  size_t lds;
};

// V: the widest access (up to 16 B) that the rotated half and half of what is not rotated are whole multiples of.
// The workgroup takes as many tokens at once as give it up to 256 lanes (a set), and a few sets per run: more sets cost
// fewer barriers, workgroups and (append) chains of loads to a token's cache row, fewer keep the chip full. Measured in
// graph replays: forward of 65,536 x 512 at two / four sets a run 74.4 / 79.6 us; append of 32 x 1024 x 256 at one / two /
// four / eight 33 / 21.1 / 19.1 / 22.1; backward of 8,192 x 256 in 512 / 1,024 workgroups 14.7 / 15.5 with its dw sum.
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
  const int64_t most = mode == MODE_APPEND ? 64 : kMaxRun;  // tokens of a run
  p.passes = (int)cdiv(ipt, kThreads);
  p.slots = p.passes > 1 ? 1 : (int)std::min<int64_t>(kThreads / ipt, most / 2);
  p.block = p.passes > 1 ? kThreads : (int)(cdiv(p.slots * ipt, 64) * 64);
  const int64_t kRuns = mode == MODE_FWD ? 2048 : mode == MODE_BWD ? 512 : 1024, kSets = mode == MODE_APPEND ? 4 : 2;
  const int64_t sets = std::max<int64_t>(1, std::min<int64_t>({kSets, most / p.slots, N / (p.slots * kRuns)}));
  p.run = (int)(p.slots * sets);
  p.grid = std::min<int64_t>(cdiv(N, p.run), mode == MODE_BWD ? 1024 : (int64_t)1 << 20);
  p.lds = 2 * hd * sizeof(float) + std::max<size_t>((size_t)p.run * R2, 8) * sizeof(float2);  // 8: see ct in the kernel
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
  a.magic_r = R ? ((1ull << 32) + R / 2 - 1) / (R / 2) : 0;
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
  dw_sum_kernel<<<(unsigned)cdiv(2 * hd, 16), 256, 0, st>>>(a.part, p.grid, (int)(2 * hd), dw);
  ESGPT_LAUNCH_CHECK();
  return ESGPT_OK;
}

int esgpt_kv_append_paged(const void* qkv, const float* q_w, const float* k_w, const void* pos, int pos_dtype,
                          const float* inv_freq, int64_t R, float eps, const uint8_t* row_mask, const int32_t* past,
                          const int32_t* page_table, int64_t table_w, void* k_pages, void* v_pages, int64_t n_pages,
                          int64_t page_size, void* q, int64_t S, int64_t Lq, int64_t H, int64_t hd, int dtype,
                          int32_t* err, void* stream) {
  // the kernel counts tokens in 32 bits, and a sequence's kept rows in f32
  constexpr int64_t kTop = ((int64_t)1 << 31) - 1024;
  ESGPT_REQUIRE(S >= 0 && Lq >= 0 && Lq <= (int64_t)1 << 24 && S <= kTop && S * Lq <= kTop);
  ESGPT_REQUIRE(rope_ok(qkv, q_w, k_w, pos, pos_dtype, inv_freq, R, S * Lq, H, hd, eps, dtype));
  ESGPT_REQUIRE(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0 && table_w >= 0 &&
                table_w < (int64_t)1 << 31 && n_pages >= 0 && n_pages < (int64_t)1 << 31);
  if (S * Lq == 0) return ESGPT_OK;
  ESGPT_REQUIRE(past && q && aligned16(q) && (table_w == 0 || page_table) &&
                (n_pages == 0 || (k_pages && v_pages && aligned16(k_pages) && aligned16(v_pages))));
  // one pool for both, or pools that overlap: keys and values would overwrite each other in no order
  const uintptr_t pool = (uintptr_t)n_pages * H * page_size * hd * (dtype == ESGPT_BF16 ? 2 : 4), kp = (uintptr_t)k_pages,
                  vp = (uintptr_t)v_pages;
  ESGPT_REQUIRE((kp < vp ? vp - kp : kp - vp) >= pool);
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
  while (((int64_t)1 << a.psl) < page_size) ++a.psl;
  launch<MODE_APPEND>(p, a, dtype, as_stream(stream));
  ESGPT_LAUNCH_CHECK();
  return ESGPT_OK;
}

}  // extern "C"
