// Attention of newly generated events over a paged cache in which n trajectories share one subject's history.
//
// generate(num_return_sequences = n) continues every subject n times from the same history. Group g's history is kept
// once (prefix pages, P_g rows); trajectory s = g n .. g n + n - 1 has its own pages (own rows). A new event i of s at
// own row t_i sees every history row and own rows <= t_i, inside the window if there is one (index distance < window):
//   o = sum_j e^{q.k_j - m} v_j / sum_j e^{q.k_j - m},  m = max_j q.k_j   (no 1/sqrt(hd), as esgpt_attn_fwd)
//
// The bound is HBM: 2 hd s bytes per history row and head ONCE per group, and the same per own row. So the rows of a
// group (n trajectories x Lq events) are the columns of one matrix product: S^T = K Q^T and O^T = V^T P^T on the 16-wide
// MFMAs, where lane l holds column (query row) l % 16 and keys 4 (l / 16) .. + 3 of a 16-key tile, so a row's softmax
// statistics are lane-local but for two lane swaps, and P goes from the accumulator to the next product's operand
// without leaving its lane. An own row is one column of sixteen: 15/16 of the MFMA rate idles there, which costs
// nothing as long as memory is the bound (a bf16 tile of 16 keys x 64 takes 96 MFMA cycles, two thirds of them for the two
// parts of P (Walk::pv), for 4 KB: 43 B per cycle and SIMD, against the 13 B per cycle that HBM gives a whole CU).
//
// Two forms (shared_plan chooses and holds the measurements). Whole: one workgroup per (group, head, 4..16 rows) does the
// history and the own rows and writes the result. Split: the history of each (group, head, 16 or 32 rows) is cut into
// chunks, one workgroup each, whose four waves take every fourth block of keys and join through LDS, and the own rows of
// each (trajectory, head) into chunks of one wave; each part leaves (m, l, O) in f32 and a second kernel joins a row's
// parts. The cut follows the caller's bounds on the lengths (the lengths themselves are on the device).
//
// A wave keeps 16 KB of keys and values in flight (Walk::pass). What it walks by is scalar: page places, ends, buffer
// descriptors. Measured with those in vector registers (a wave's number taken from threadIdx, a length loaded like data),
// every buffer load became a loop over the lanes: 3,555 vector instructions a wave against 1,622, 32 x 16 over 256 + 64
// events 15.5 us against 13.1; 64 keys a block rather than 32, 8 x 32 over 16,384 events 59.5 -> 58.9 at 512 chunks.
// Now 8 x 32 over 16,384 + 64 (hd 64, 8 heads, bf16) takes 54 us + 5 of join: 4.8 TB/s, a
// large copy reaches 4.95.
//
// Nothing is read beyond a sequence's length: rows past it are zeros in registers, so what an unused part of a page
// holds (NaN, infinity) never meets a product. Where a tile is partly masked (a window's edge, a later event of the same
// call), 0 x infinity is kept out of the other rows by an exact second pass (masked_pv).
#include "common.h"

#include <algorithm>

using namespace esgpt;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kMaxLq = 16;
constexpr float kLog2e = 1.44269504088896340736f;

struct SharedArgs {
  const void *q, *kp, *vp;
  void* o;
  const int32_t *prefix_table, *prefix_lens, *table, *past;
  const uint8_t* row_mask;  // [S, Lq] or null
  float* ml;                // [S Lq H, NP, 2] (m, l)
  float* po;                // [S Lq H, NP, hd]
  int32_t* err;
  int64_t n_pages, prefix_w, table_w;
  int S, n, Lq, H, hd, psl;     // psl: log2 of the page size
  int prefix_cap, cap;
  int window, owin;             // the window where it can cut the history, the own rows (0: never)
  uint32_t far;                 // the window of a row beyond the cap
  int M, RT, tr;                // rows of a group; row tiles of the history's workgroups; whole form: rows of a tile
  int NPc, NSc, NP, pchunk, schunk;
  int units;  // history workgroups; the own rows' follow
};

__device__ __forceinline__ float xmax(float v) {  // over the four lanes of one column
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float xsum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// e^{s - m}, m >= s the running maximum (0 while there is none). The difference comes first: it is exact near the maximum,
// where s log2(e) - (m log2(e) rounded) would be off by 2^-24 of m, a factor beyond f32 for scores above 10^9.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float weight(float s, float base) { return __builtin_amdgcn_exp2f((s - base) * kLog2e); }
// A value that is the same in every lane, in a scalar register: buffer descriptors, page places and loop bounds that the
// compiler finds in vector registers cost a loop over the lanes at each use.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Smallest / largest value over the sixteen columns (a column's four lanes hold the same), as a scalar.
template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false); }
__device__ __forceinline__ int cols_min(int v) {
  v = min(v, dpp_i<0xB1>(v));
  v = min(v, dpp_i<0x4E>(v));
  v = min(v, dpp_i<0x141>(v));
  v = min(v, dpp_i<0x140>(v));
  return scalar(v);
}
__device__ __forceinline__ int cols_max(int v) { return -cols_min(-v); }

// One new event: its place among its trajectory's own rows. active: it exists, is not padding and its past is sane.
struct Row {
  uint32_t at;  // own row
  bool far;     // it lies beyond the cap: a window still counts from it
  bool active;
};
__device__ __forceinline__ Row row_of(const SharedArgs& a, int s, int i, bool exists) {
  Row r{0, false, false};
  if (!exists) return r;
  const int past = a.past[s];
  int k = i;
  bool keep = true;
  if (a.row_mask) {
    k = 0;
    for (int j = 0; j < i; ++j) k += a.row_mask[(int64_t)s * a.Lq + j] != 0;
    keep = a.row_mask[(int64_t)s * a.Lq + i] != 0;
  }
  if (!keep) return r;
  r.far = past > a.cap - 1 - k;
  if (past < 0 || r.far) {  // a row that the cache has no place for
    set_err(a.err, ESGPT_FLAG_BAD_PAGE);
    if (past < 0) return r;
  }
  r.at = (uint32_t)past + k;
  r.active = true;
  return r;
}
// How many of the first `end` rows lie before the window of the row that has n - 1 rows before it, and how many up to it.
__device__ __forceinline__ int rows_before(const SharedArgs& a, const Row& r, uint32_t n, int window, int end) {
  const uint32_t w = r.far ? a.far : window ? (uint32_t)window : ~0u;
  return (int)min((uint32_t)end, n - min(n, w));
}
__device__ __forceinline__ int rows_to(uint32_t n, int end) { return (int)min((uint32_t)end, n); }
__device__ __forceinline__ int prefix_len(const SharedArgs& a, int g) {
  if (a.prefix_cap == 0) return 0;
  const int P = a.prefix_lens[g];
  if (P < 0 || P > a.prefix_cap) set_err(a.err, ESGPT_FLAG_BAD_PAGE);
  return scalar(min(max(P, 0), a.prefix_cap));
}

// Dimension of accumulator register r of tile dt in lane group g (= lane / 16). bf16: the transposed V tile's natural
// rows. f32: tiles 2p and 2p + 1 hold the even and odd dimensions of 32p .. 32p + 31, so that a lane reads V in pairs.
template <typename T>
__device__ __forceinline__ int dim_of(int dt, int g, int r) {
  if constexpr (sizeof(T) == 2) return 16 * dt + 4 * g + r;
  else return 32 * (dt >> 1) + 2 * (4 * g + r) + (dt & 1);
}

// Four neighbouring dimensions dim .. dim + 3 of one column: of tile d in bf16; in f32, registers 2 (d & 1) and
// 2 (d & 1) + 1 of the pair of tiles that d belongs to.
template <typename T, int DT>
__device__ __forceinline__ float4 four(const f32x4 (&acc)[DT], int d, int g, int& dim) {
  if constexpr (sizeof(T) == 2) {
    dim = 16 * d + 4 * g;
    return make_float4(acc[d][0], acc[d][1], acc[d][2], acc[d][3]);
  } else {
    const int p = d & ~1, r = 2 * (d & 1);
    dim = 16 * p + 8 * g + 2 * r;
    return make_float4(acc[p][r], acc[p + 1][r], acc[p][r + 1], acc[p + 1][r + 1]);
  }
}

// The online softmax of NT x 16 rows: O^T tiles (column = row of q), running maximum, this lane's share of the sum.
template <int NT, int DT>
struct State {
  f32x4 acc[NT][DT];
  float m[NT], l[NT];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// One wave's walk over blocks of keys.
template <typename T, int KD>
struct Walk {
  static constexpr bool kBf16 = sizeof(T) == 2;
  // 16-key tiles per block: 16 KB of keys and values per block and wave at 64 dimensions and at 128 in bf16
  static constexpr int KT = kBf16 ? (KD <= 2 ? 4 : 2) : (KD <= 2 ? 2 : 1);
  static constexpr int KB = 16 * KT;
  static constexpr int DT = 2 * KD;        // 16-wide tiles of the head
  static constexpr int LD = KD * 32 + 16;  // LDS row of V (elements): 8 mod 16 dwords, transposed reads hit all banks
  static constexpr int NK = kBf16 ? KD : 2 * KD;     // 16-B chunks of a key, or of a query, that a lane holds
  static constexpr int LPR = KD == 3 ? 16 : 4 * KD;  // bf16: lanes that read one row of V (12 of 16 at 96)
  static constexpr int VT = kBf16 ? LPR / 4 : 2 * KD;  // 16-B loads (f32: register groups) of a tile's V
  static constexpr int NV = KT * VT;
  static constexpr int PER = 64 / KT;                  // blocks whose page ids one load brings
  static constexpr int kOut = 1 << 30;
  using Q = uint4[NK];

  const SharedArgs& a;
  int h, lane, g, c;  // g = lane / 16, c = lane % 16
  __bf16* vt;         // bf16: this wave's V tile, KB x LD
  // Byte offsets of this lane's chunks in a 16-row tile; beyond the head's width: out of every range (reads zero).
  int ko[NK], vo[kBf16 ? 1 : KD];

  __device__ __forceinline__ Walk(const SharedArgs& a_, int h_, void* lds) : a(a_), h(h_) {
    lane = lane_id();
    g = lane >> 4;
    c = lane & 15;
    vt = reinterpret_cast<__bf16*>(lds);
    constexpr int E = kBf16 ? 8 : 4;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int d = k * 4 * E + E * g;
      ko[k] = d < a.hd ? (c * a.hd + d) * (int)sizeof(T) : kOut;
    }
    if constexpr (kBf16) {
      const int d = (lane % LPR) * 8;
      vo[0] = d < a.hd ? (lane / LPR * a.hd + d) * 2 : kOut;
    } else {
#pragma unroll
      for (int p = 0; p < KD; ++p) {
        const int d = 32 * p + 2 * c;
        vo[p] = d < a.hd ? (4 * g * a.hd + d) * 4 : kOut;
      }
    }
  }

  // Queries: column c is row `out` of q. bf16: chunk k holds dims 32 k + 8 g .. + 7; f32: dims 16 k + 4 g .. + 3 (the
  // products contract over lane groups, in this permuted order on both sides).
  __device__ __forceinline__ void load_q(Q& qf, int64_t out, bool exists) const {
    constexpr int E = kBf16 ? 8 : 4;
    const T* p = reinterpret_cast<const T*>(a.q) + (out * a.H + h) * a.hd;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int d = k * 4 * E + E * g;
      qf[k] = (exists && d < a.hd) ? *reinterpret_cast<const uint4*>(p + d) : make_uint4(0, 0, 0, 0);
    }
  }

  // Page ids of the 64 / KT blocks from k0 on, one lane each, for keys below `limit` (a bound that needs no length to
  // have arrived); -1 beyond. check(): what the walk up to k_end uses of them.
  __device__ __forceinline__ int key_of(int k0, int stride) const { return k0 + (lane / KT) * stride + (lane % KT) * 16; }
  __device__ __forceinline__ int pages(const int32_t* tab, int k0, int stride, int limit) const {
    const int key = key_of(k0, stride);
    return k0 >= 0 && key < limit ? tab[key >> a.psl] : -1;
  }
  // Byte offsets of the pages' rows that a walk up to k_end reads, worked out for all lanes at once; hi < 0: none.
  struct Offsets {
    int lo, hi;
  };
  __device__ __forceinline__ Offsets check(int id, int k0, int stride, int k_end) const {
    const int key = key_of(k0, stride);
    if (key >= k_end) return {0, -1};
    if (id < 0 || id >= a.n_pages) {
      set_err(a.err, ESGPT_FLAG_BAD_PAGE);
      return {0, -1};
    }
    const int64_t off = ((((int64_t)id * a.H + h) << a.psl) + (key & ((1 << a.psl) - 1))) * (a.hd * (int)sizeof(T));
    return {(int)off, (int)(off >> 32)};
  }

  // A block's 16-row tiles: where they are in the pools and how many bytes of them a walk may read (none on a bad page).
  struct Tiles {
    int64_t off[KT];
    int bytes[KT];
  };
  __device__ __forceinline__ Tiles tiles(int k0, int k_end, const Offsets& of, int slot) const {
    Tiles b;
    const int rb = a.hd * (int)sizeof(T);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int hi = __builtin_amdgcn_readlane(of.hi, slot * KT + t);
      const uint32_t lo = __builtin_amdgcn_readlane(of.lo, slot * KT + t);
      b.off[t] = (int64_t)scalar(max(hi, 0)) << 32 | (uint32_t)scalar((int)lo);
      b.bytes[t] = scalar(hi >= 0 ? min(16, max(0, k_end - k0 - 16 * t)) * rb : 0);
    }
    return b;
  }
  // Range-checked buffers: rows past the end read as zeros.
  __device__ __forceinline__ static __amdgpu_buffer_rsrc_t rows(const void* pool, int64_t off, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(reinterpret_cast<const char*>(pool) + off), (short)0, bytes,
                                             0x00020000);
  }
  __device__ __forceinline__ void load_k(uint4 (&k)[KT * NK], const Tiles& b) const {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const __amdgpu_buffer_rsrc_t r = rows(a.kp, b.off[t], b.bytes[t]);
#pragma unroll
      for (int i = 0; i < NK; ++i)
        k[t * NK + i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, ko[i], 0, 0));
    }
  }
  __device__ __forceinline__ void load_v(uint4 (&v)[NV], const Tiles& b) const {
    const int rb = a.hd * (int)sizeof(T);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const __amdgpu_buffer_rsrc_t r = rows(a.vp, b.off[t], b.bytes[t]);
      if constexpr (kBf16) {
#pragma unroll
        for (int i = 0; i < VT; ++i)
          v[t * VT + i] =
              __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, vo[0] + i * (64 / LPR) * rb, 0, 0));
      } else {
        float2* f = reinterpret_cast<float2*>(v + t * VT);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int p = 0; p < KD; ++p)
            f[e * KD + p] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, vo[p] + e * rb, 0, 0));
      }
    }
  }

  // O += P.V of one block whose V tile is in LDS, P as the sum of two bf16: its upper half and what that leaves (off by
  // 2^-15 of P; the 2^-20 keep the second part above zero while P > 2^-106, so that a visible infinity stays one). One
  // part alone, off by 2^-8, is as coarse as the output's own rounding: 32 x 16 over 256 + 64 was off by 1.78e-3 of the
  // result, the plain form in f32 by 1.66e-3. The second costs three vector operations a probability and as many products
  // as the first: 11.4 -> 11.8 us there, 55.8 -> 56.4 over 8 x 32, 16,384 + 64.
  template <int NT>
  __device__ __forceinline__ void pv(State<NT, DT>& st, const float (&p)[NT][4 * KT]) const {
    const __bf16* vr = vt + (4 * g + (c >> 2)) * LD + 4 * (c & 3);
#pragma unroll
    for (int u = 0; u < KT; u += 2) {
      bf16x8 ph[NT], pl[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float pi = p[t][4 * u + i];
          const uint32_t hi = __float_as_uint(pi) & 0xFFFF0000u;
          ph[t][i] = __builtin_bit_cast(__bf16, (uint16_t)(hi >> 16));
          pl[t][i] = (__bf16)fmaf(pi, 1.f + 0x1p-20f, -__uint_as_float(hi));
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        typedef __attribute__((address_space(3))) bf16x4* lds4;
        const bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(vr + 16 * u * LD + 16 * d));
        const bf16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(vr + 16 * (u + 1) * LD + 16 * d));
        bf16x8 vf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          vf[i] = x[i];
          vf[4 + i] = y[i];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          st.acc[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph[t], st.acc[t][d], 0, 0, 0);
          st.acc[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[t], st.acc[t][d], 0, 0, 0);
        }
      }
    }
  }

  // P.V of a partly masked block key by key: a key adds nothing (not even 0 x infinity) to the rows
  // that do not see it. Reads the values again; only a walk that has met a value that is not finite comes here.
  __device__ __forceinline__ void masked_pv(const Offsets& of, int slot, const float (&p)[4 * KT], f32x4 (&o)[DT], int k0,
                                            int lo, int hi) const {
#pragma nounroll
    for (int i = 0; i < 4 * KT; ++i) {
      const int oh = __builtin_amdgcn_readlane(of.hi, slot * KT + (i >> 2));
      if (oh < 0) continue;
      const uint32_t ol = __builtin_amdgcn_readlane(of.lo, slot * KT + (i >> 2));
      const T* vb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.vp) + ((int64_t)oh << 32 | ol));
      float pi = p[0];
#pragma unroll
      for (int j = 1; j < 4 * KT; ++j) pi = i == j ? p[j] : pi;
#pragma nounroll
      for (int gg = 0; gg < 4; ++gg) {
        const float pk = __shfl(pi, 16 * gg + c, 64);
        const int row = 4 * gg + (i & 3), key = k0 + (i & ~3) * 4 + row;
        if (key < lo || key >= hi) continue;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int dim = dim_of<T>(d, g, x);
            if (dim < a.hd) o[d][x] = fmaf(pk, to_f32(vb[row * a.hd + dim]), o[d][x]);
          }
      }
    }
  }

  // A place in a walk: block k0 of segment seg, whose rows end at k_end; of: page offsets of the round of blocks that
  // slot counts in.
  struct At {
    int seg, k0, k_end, slot;
    Offsets of;
  };
  // Opens the first segment from `seg` on that has a key; false: none is left.
  template <class Segs>
  __device__ __forceinline__ bool open(Segs& sg, int seg, At& at) const {
    for (; seg < sg.count; ++seg) {
      int raw;
      sg.open(*this, seg, at.k0, at.k_end, raw);
      at.k0 = scalar(at.k0);
      at.k_end = scalar(at.k_end);
      if (at.k0 >= at.k_end) continue;
      at.seg = seg;
      at.slot = 0;
      at.of = check(raw, at.k0, sg.stride(seg), at.k_end);
      return true;
    }
    return false;
  }
  template <class Segs>
  __device__ __forceinline__ bool next(Segs& sg, At& at) const {
    const int stride = sg.stride(at.seg), k1 = at.k0 + stride;
    if (k1 >= at.k_end) return open(sg, at.seg + 1, at);
    at.k0 = k1;
    if (++at.slot == PER) {
      at.slot = 0;
      at.of = check(pages(sg.table(at.seg), k1, stride, at.k_end), k1, stride, at.k_end);
    }
    return true;
  }

  // One pass over the segments of Segs (runs of keys with one page table and one set of limits each: row (column c of
  // tile t) sees keys [lo[t], hi[t])), block by block. A block's V goes to LDS at the top of its step and its K to the
  // matrix units right after, and the next block's loads (of the next segment, at a segment's end) follow each: one set
  // of registers, a whole step of latency covered.
  // exact: see masked_pv.
  template <int NT, class Segs>
  __device__ __forceinline__ void pass(State<NT, DT>& st, const Q (&qf)[NT], Segs& sg, bool exact) const {
    At at;
    if (!open(sg, 0, at)) return;
    Tiles nb = tiles(at.k0, at.k_end, at.of, 0);
    uint4 k[KT * NK], v[NV];
    load_k(k, nb);
    load_v(v, nb);
    int lo[NT], hi[NT], lo_all, hi_all, seg = -1;
    for (;;) {
      const At now = at;
      const int k0 = at.k0;
      uint32_t gone = 0;  // tiles without a row: a bad page, or past the end
#pragma unroll
      for (int t = 0; t < KT; ++t) gone |= nb.bytes[t] == 0 ? 1u << t : 0u;
      if (seg != at.seg) sg.limits(seg = at.seg, lo, hi, lo_all, hi_all);
      const bool more = next(sg, at);
      if (more) nb = tiles(at.k0, at.k_end, at.of, at.slot);
      const bool full = k0 >= lo_all && k0 + KB <= hi_all && k0 + KB <= now.k_end && !gone;
      if constexpr (kBf16) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int row = i * (64 / LPR) + lane / LPR, d = (lane % LPR) * 8;
          if (KD != 3 || d < 32 * KD) *reinterpret_cast<uint4*>(vt + row * LD + d) = v[i];
        }
        if (more) load_v(v, nb);
      }
      f32x4 s[NT][KT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
          if constexpr (kBf16) {
#pragma unroll
            for (int i = 0; i < KD; ++i)
              s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[u * KD + i]),
                                                                __builtin_bit_cast(bf16x8, qf[t][i]), s[t][u], 0, 0, 0);
          } else {
#pragma unroll
            for (int i = 0; i < 2 * KD; ++i) {
              const f32x4 kf = __builtin_bit_cast(f32x4, k[u * NK + i]), q4 = __builtin_bit_cast(f32x4, qf[t][i]);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], q4[e], s[t][u], 0, 0, 0);
            }
          }
        }
      if (more) load_k(k, nb);
      float p[NT][4 * KT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (!full) {
          // a masked score is -inf (it may be NaN); its probability is then an exact zero
          const int l0 = lo[t] - k0 - 4 * g;
          const uint32_t span = (uint32_t)max(hi[t] - lo[t], 0);
#pragma unroll
          for (int u = 0; u < KT; ++u) {
            const uint32_t su = gone >> u & 1 ? 0u : span;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!((uint32_t)(16 * u + r - l0) < su)) s[t][u][r] = -INFINITY;
          }
        }
        float mx = s[t][0][0];
#pragma unroll
        for (int i = 1; i < 4 * KT; ++i) mx = fmaxf(mx, s[t][i >> 2][i & 3]);
        const float mn = fmaxf(st.m[t], xmax(mx));
        const float mc = base_of(mn);
        if (__any(mn != st.m[t])) {
          const float f = weight(st.m[t], mc);
          st.l[t] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) st.acc[t][d] *= f;
          st.m[t] = mn;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * KT; ++i) {
          p[t][i] = weight(s[t][i >> 2][i & 3], mc);
          sum += p[t][i];
        }
        st.l[t] += sum;
      }
      if (exact && !full) {
#pragma unroll
        for (int t = 0; t < NT; ++t) masked_pv(now.of, now.slot, p[t], st.acc[t], k0, lo[t], hi[t]);
      } else if constexpr (kBf16) {
        pv(st, p);
      } else {
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          const float* f = reinterpret_cast<const float*>(v + u * VT);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int t = 0; t < NT; ++t)
                st.acc[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[(e * KD + (d >> 1)) * 2 + (d & 1)], p[t][4 * u + e],
                                                                    st.acc[t][d], 0, 0, 0);
        }
      }
      if (!more) break;
      if constexpr (!kBf16) load_v(v, nb);
    }
  }

  // A pass; where a sum is not finite, another that keeps such values from the rows that do not see them (0 x infinity
  // would have reached the whole block's).
  template <int NT, class Segs>
  __device__ __forceinline__ void walk(State<NT, DT>& st, const Q (&qf)[NT], const Segs& segments) const {
    for (bool exact = false;; exact = true) {
      st.clear();
      Segs sg = segments;
      pass(st, qf, sg, exact);
      if (exact) return;
      float z = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) z = fmaf(st.acc[t][d][r], 0.f, z);
      if (!__any(z != 0.f)) return;
    }
  }
};

// v / l, zeros for a row that saw no key (l == 0; what v holds then does not count).
template <typename T>
__device__ __forceinline__ void store4(T* o, float4 v, float l) {
  const bool none = l == 0.f;
  const float inv = 1.f / l;
  struct alignas(4 * sizeof(T)) Four { T e[4]; } x;
  x.e[0] = from_f32<T>(none ? 0.f : v.x * inv);
  x.e[1] = from_f32<T>(none ? 0.f : v.y * inv);
  x.e[2] = from_f32<T>(none ? 0.f : v.z * inv);
  x.e[3] = from_f32<T>(none ? 0.f : v.w * inv);
  *reinterpret_cast<Four*>(o) = x;
}

// A part's result of one row: stored for the join, or, as the only part, divided and written to o.
template <typename T>
__device__ __forceinline__ void emit4(const SharedArgs& a, int64_t out, int h, int part, int d, float4 v, float m, float l,
                                      bool first) {
  const int64_t rh = out * a.H + h;
  if (a.NP == 1) {
    store4(reinterpret_cast<T*>(a.o) + rh * a.hd + d, v, l);
    return;
  }
  const int64_t at = rh * a.NP + part;
  if (first) *reinterpret_cast<float2*>(a.ml + 2 * at) = make_float2(m, l);
  if (l != 0.f) *reinterpret_cast<float4*>(a.po + at * a.hd + d) = v;  // l == 0: the join does not read it
}

// The waves' states of one tile of 16 rows, joined per row through LDS, 64 dimensions at a time: row r0 + i of the group
// is column i < n. Every thread of the workgroup calls this.
template <typename T, int KD, int NW>
struct Join {
  static constexpr int W = KD * 32 < 64 ? KD * 32 : 64, OLD = W + 4;
  static constexpr int kBytes = NW * 16 * (OLD + 2) * 4;
  template <int NT>
  __device__ __forceinline__ static void run(const SharedArgs& a, const State<NT, 2 * KD>& st, int t, bool act, char* lds,
                                             int64_t out0, int r0, int n, int h, int part) {
    const int w = scalar(threadIdx.x >> 6), lane = lane_id(), g = lane >> 4, c = lane & 15;
    float* jo = reinterpret_cast<float*>(lds);  // [wave][16][OLD]
    float* jm = jo + NW * 16 * OLD;             // [wave][16]
    float* jl = jm + NW * 16;
    const float lw = act ? xsum(st.l[t]) : 0.f;
    const int row = threadIdx.x >> 4;
    const bool mine = row < n && r0 + row < a.M;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int d0 = 0; d0 < KD * 32; d0 += W) {
      __syncthreads();  // the waves' V tiles, or the reads of the round before
      if (d0 == 0 && g == 0) {
        jm[w * 16 + c] = st.m[t];
        jl[w * 16 + c] = lw;
      }
#pragma unroll
      for (int d = 0; d < 2 * KD; ++d) {
        int dim;
        const float4 v = four<T, 2 * KD>(st.acc[t], d, g, dim);
        if (d / (W / 16) == d0 / W) *reinterpret_cast<float4*>(jo + (w * 16 + c) * OLD + dim - d0) = v;
      }
      __syncthreads();
      if (!mine) continue;
      if (d0 == 0) {
        for (int u = 0; u < NW; ++u) M = fmaxf(M, jl[u * 16 + row] == 0.f ? -INFINITY : jm[u * 16 + row]);
      }
      const float mc = base_of(M);
      const int d = d0 + 4 * (threadIdx.x & 15);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float Ls = 0.f;
      for (int u = 0; u < NW; ++u) {
        const float lu = jl[u * 16 + row];
        if (lu == 0.f) continue;  // this wave saw nothing for the row
        const float f = weight(jm[u * 16 + row], mc);
        Ls = fmaf(lu, f, Ls);
        if (d - d0 >= W) continue;
        const float4 y = *reinterpret_cast<const float4*>(jo + (u * 16 + row) * OLD + d - d0);
        v.x = fmaf(y.x, f, v.x);
        v.y = fmaf(y.y, f, v.y);
        v.z = fmaf(y.z, f, v.z);
        v.w = fmaf(y.w, f, v.w);
      }
      if (d0 == 0) L = Ls;
      if (d - d0 < W && d < a.hd) emit4<T>(a, out0 + r0 + row, h, part, d, v, M, L, d == 0);
    }
  }
};

// The limits that hold for every column that counts: blocks within them need no mask.
template <int NT>
__device__ __forceinline__ void common_limits(const int (&lo)[NT], const int (&hi)[NT], const bool (&act)[NT], int& lo_all,
                                              int& hi_all) {
  lo_all = 0;
  hi_all = 0x7fffffff;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (act[t]) {
      lo_all = max(lo_all, lo[t]);
      hi_all = min(hi_all, hi[t]);
    }
  lo_all = cols_max(lo_all);
  hi_all = cols_min(hi_all);
}

// One segment: a chunk of a history, or of one trajectory's own rows.
template <int NT>
struct OneSegment {
  const int32_t* tab;
  int first, end, step, raw, lo[NT], hi[NT];
  bool act[NT];
  static constexpr int count = 1;
  __device__ __forceinline__ int stride(int) const { return step; }
  __device__ __forceinline__ const int32_t* table(int) const { return tab; }
  template <class W>
  __device__ __forceinline__ void open(const W&, int, int& k0, int& k_end, int& ids) const {
    k0 = first;
    k_end = end;
    ids = raw;
  }
  __device__ __forceinline__ void limits(int, int (&l)[NT], int (&u)[NT], int& lo_all, int& hi_all) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] = lo[t];
      u[t] = hi[t];
    }
    common_limits<NT>(lo, hi, act, lo_all, hi_all);
  }
};

// Split form: a workgroup per history chunk of one (group, head, 16 NT rows), then four waves a workgroup with the own
// rows of one (trajectory, head, chunk) each.
template <typename T, int KD, int NT>
__global__ __launch_bounds__(64 * kWaves, KD * NT < 8 ? 2 : 1) void shared_kernel(SharedArgs a) {
  using W = Walk<T, KD>;
  using J = Join<T, KD, kWaves>;
  constexpr int kTile = W::kBf16 ? W::KB * W::LD * 2 : 0;
  __shared__ __align__(16) char lds[(kWaves * kTile > J::kBytes) ? kWaves * kTile : J::kBytes];
  const int w = scalar(threadIdx.x >> 6), lane = lane_id(), g = lane >> 4, c = lane & 15;

  if ((int)blockIdx.x >= a.units) {
    // column c is the trajectory's new event c
    const int id = (int)(blockIdx.x - a.units) * kWaves + w;
    const int ch = id % a.NSc, sh = id / a.NSc, h = sh % a.H, s = sh / a.H;
    if (s >= a.S) return;
    // a bound of 0 leaves no history workgroup to see a length beyond it
    if (a.units == 0 && a.prefix_lens && a.prefix_lens[s / a.n] != 0) set_err(a.err, ESGPT_FLAG_BAD_PAGE);
    const W x(a, h, lds + w * kTile);
    OneSegment<1> sg;
    sg.tab = a.table + (int64_t)s * a.table_w;
    sg.step = W::KB;
    sg.raw = a.owin ? -1 : x.pages(sg.tab, ch * a.schunk, W::KB, a.cap);
    typename W::Q q[1];
    x.load_q(q[0], (int64_t)s * a.Lq + c, c < a.Lq);
    const Row r = row_of(a, s, c, c < a.Lq);
    sg.act[0] = r.active;
    sg.hi[0] = r.active ? rows_to(r.at + 1, a.cap) : 0;
    sg.lo[0] = r.active ? rows_before(a, r, r.at + 1, a.owin, a.cap) : 0;
    const int base = a.owin ? cols_min(r.active ? sg.lo[0] : a.cap) & ~15 : 0;
    const int end = cols_max(sg.hi[0]);  // no active row: no key
    sg.first = base + ch * a.schunk;
    sg.end = min(end, sg.first + a.schunk);
    if (a.owin && sg.first < sg.end) sg.raw = x.pages(sg.tab, sg.first, W::KB, sg.end);
    State<1, W::DT> st;
    x.walk(st, q, sg);
    const float l = r.active ? xsum(st.l[0]) : 0.f;
    if (c < a.Lq) {
#pragma unroll
      for (int d = 0; d < W::DT; ++d) {
        int dim;
        const float4 v = four<T, W::DT>(st.acc[0], d, g, dim);
        if (dim < a.hd) emit4<T>(a, (int64_t)s * a.Lq + c, h, a.NPc + ch, dim, v, st.m[0], l, d == 0 && g == 0);
      }
    }
    return;
  }

  // neighbouring workgroups of one XCD share a chunk's keys and values
  const int id = xcd_linear(blockIdx.x, a.units);
  const int rt = id % a.RT, ch = id / a.RT % a.NPc, gh = id / a.RT / a.NPc;
  const int h = gh % a.H, grp = gh / a.H;
  const int64_t out0 = (int64_t)grp * a.M;
  const W x(a, h, lds + w * kTile);
  OneSegment<NT> sg;
  sg.tab = a.prefix_table + (int64_t)grp * a.prefix_w;
  sg.step = kWaves * W::KB;
  sg.raw = a.window ? -1 : x.pages(sg.tab, ch * a.pchunk + w * W::KB, sg.step, a.prefix_cap);
  typename W::Q q[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int rr = rt * 16 * NT + 16 * t + c;
    x.load_q(q[t], out0 + rr, rr < a.M);
  }
  const int P = prefix_len(a, grp);
  int base = a.prefix_cap;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int rr = rt * 16 * NT + 16 * t + c;
    const Row r = row_of(a, grp * a.n + rr / a.Lq, rr % a.Lq, rr < a.M);
    sg.act[t] = r.active;
    sg.hi[t] = r.active ? P : 0;
    sg.lo[t] = r.active ? rows_before(a, r, P + r.at + 1, a.window, P) : 0;
    if (r.active) base = min(base, sg.lo[t]);
  }
  // chunks count from the first row that a window of this group can reach, whatever its own rows
  const int c0 = ((a.window ? max(0, P - a.window) : 0) & ~15) + ch * a.pchunk;
  sg.end = min(P, c0 + a.pchunk);
  sg.first = c0 + w * W::KB;
  if (a.window) {  // whole rounds of blocks before the first visible key
    sg.first += max(0, (cols_min(base) & ~15) - c0) / sg.step * sg.step;
    if (sg.first < sg.end) sg.raw = x.pages(sg.tab, sg.first, sg.step, sg.end);
  }
  State<NT, W::DT> st;
  x.walk(st, q, sg);
  J::run(a, st, 0, sg.act[0], lds, out0, rt * 16 * NT, 16, h, ch);
  if constexpr (NT == 2) J::run(a, st, 1, sg.act[1], lds, out0, rt * 16 * NT + 16, 16, h, ch);
}

// Whole form: one workgroup of NW waves per (group, head, `tr` rows) does the rows' history and their own rows and writes
// the result. The waves take every NW-th block of the history (segment 0) and, from the other end, every NW-th
// trajectory's own rows, which only that trajectory's columns see; a segment's page ids are loaded when the one before is
// opened.
//
// Four waves (above 64 dimensions): two workgroups a CU, at most 256 registers. Left to itself f32 at 128 dimensions took 292,
// and one workgroup a CU: 16 x 64 over 1,000 + 20, 8 heads, 110 us against 79.
template <typename T, int KD, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void shared_whole_kernel(SharedArgs a) {
  using W = Walk<T, KD>;
  using J = Join<T, KD, NW>;
  constexpr int kTile = W::kBf16 ? W::KB * W::LD * 2 : 0;
  __shared__ __align__(16) char lds[(NW * kTile > J::kBytes) ? NW * kTile : J::kBytes];
  const int w = scalar(threadIdx.x >> 6), lane = lane_id(), c = lane & 15;
  const int id = xcd_linear(blockIdx.x, gridDim.x);
  const int rt = id % a.RT, gh = id / a.RT, h = gh % a.H, grp = gh / a.H;
  const int64_t out0 = (int64_t)grp * a.M;
  const W x(a, h, lds + w * kTile);

  struct Segs {
    const SharedArgs& a;
    const int32_t* ptab;
    int w, s0, count, P, my, plo, phi, olo, ohi, ids;
    int pfrom, ofrom;  // where a walk begins: no later than where the page ids that it was given do
    bool act;
    __device__ __forceinline__ int seq(int seg) const { return s0 + (NW - 1 - w) + (seg - 1) * NW; }
    __device__ __forceinline__ int stride(int seg) const { return seg == 0 ? NW * W::KB : W::KB; }
    __device__ __forceinline__ const int32_t* table(int seg) const {
      return seg == 0 ? ptab : a.table + (int64_t)seq(seg) * a.table_w;
    }
    __device__ __forceinline__ void open(const W& x, int seg, int& k0, int& k_end, int& raw) {
      raw = ids;
      if (seg == 0) {
        k0 = w * W::KB + (cols_min(act ? pfrom : P + 15) & ~15);  // no active row: no key
        k_end = P;
      } else {
        const bool mine = act && my == seq(seg);
        k0 = cols_min(mine ? ofrom : a.cap) & ~15;
        k_end = cols_max(mine ? ohi : 0);
      }
      if (seg == 0 ? a.window : a.owin) {
        if (k0 < k_end) raw = x.pages(table(seg), k0, stride(seg), k_end);
      }
      if (!a.owin && seg + 1 < count) ids = x.pages(table(seg + 1), 0, W::KB, a.cap);
    }
    __device__ __forceinline__ void limits(int seg, int (&lo)[1], int (&hi)[1], int& lo_all, int& hi_all) const {
      if (seg == 0) {
        lo[0] = plo;
        hi[0] = phi;
        const bool on[1] = {act};
        common_limits<1>(lo, hi, on, lo_all, hi_all);
      } else {  // the other trajectories' columns see none of these rows
        const bool mine = act && my == seq(seg);
        lo[0] = olo;
        hi[0] = mine ? ohi : 0;
        lo_all = hi_all = 0;
      }
    }
  };

  const int rr = rt * a.tr + c, s0 = grp * a.n + rt * a.tr / a.Lq;
  const int ns = grp * a.n + min(a.M, rt * a.tr + a.tr) / a.Lq - s0 + (min(a.M, rt * a.tr + a.tr) % a.Lq != 0);
  const bool exists = c < a.tr && rr < a.M;
  Segs sg{a, a.prefix_table + (int64_t)grp * a.prefix_w, w, s0, 1 + max(0, (ns - (NW - 1 - w) + NW - 1) / NW)};
  sg.ids = a.window ? -1 : x.pages(sg.ptab, w * W::KB, sg.stride(0), a.prefix_cap);
  typename W::Q q[1];
  x.load_q(q[0], out0 + rr, exists);
  sg.P = prefix_len(a, grp);
  sg.my = grp * a.n + rr / a.Lq;  // this column's trajectory
  const Row r = row_of(a, sg.my, rr % a.Lq, exists);
  sg.act = r.active;
  sg.phi = r.active ? sg.P : 0;
  sg.plo = r.active ? rows_before(a, r, sg.P + r.at + 1, a.window, sg.P) : 0;
  sg.ohi = r.active ? rows_to(r.at + 1, a.cap) : 0;
  sg.olo = r.active ? rows_before(a, r, r.at + 1, a.owin, a.cap) : 0;
  sg.pfrom = a.window ? sg.plo : 0;
  sg.ofrom = a.owin ? sg.olo : 0;
  State<1, W::DT> st;
  x.walk(st, q, sg);
  J::run(a, st, 0, r.active, lds, out0, rt * a.tr, a.tr, h, 0);
}

// Joins a row's parts: o = sum_p e^{m_p - M} O_p / sum_p e^{m_p - M} l_p. One wave per (row, head): lane groups of
// `width` lanes (4 dimensions each) take every (64 / width)-th part.
template <typename T>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a, int64_t rows, int width) {
  const int64_t rh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (rh >= rows) return;
  const int lane = lane_id(), sub = lane / width, d = 4 * (lane % width), nsub = 64 / width;
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + rh * a.NP;
  const float2 own = lane < a.NP ? ml[lane] : make_float2(-INFINITY, 0.f);  // NP <= 64
  const float M = wave_max(own.y == 0.f ? -INFINITY : own.x);
  const float mc = base_of(M);
  const float f = own.y == 0.f ? 0.f : weight(own.x, mc);
  const float L = wave_sum(own.y == 0.f ? 0.f : own.y * f);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < a.NP; p0 += nsub) {
    const int p = p0 + sub;
    const float fp = __shfl(f, p & 63, 64), lp = __shfl(own.y, p & 63, 64);
    if (p < a.NP && lp != 0.f && d < a.hd) {
      const float4 y = *reinterpret_cast<const float4*>(a.po + (rh * a.NP + p) * a.hd + d);
      v.x = fmaf(y.x, fp, v.x);
      v.y = fmaf(y.y, fp, v.y);
      v.z = fmaf(y.z, fp, v.z);
      v.w = fmaf(y.w, fp, v.w);
    }
  }
  for (int o = width; o < 64; o <<= 1) {
    v.x += __shfl_xor(v.x, o, 64);
    v.y += __shfl_xor(v.y, o, 64);
    v.z += __shfl_xor(v.z, o, 64);
    v.w += __shfl_xor(v.w, o, 64);
  }
  if (sub == 0 && d < a.hd) {
    store4(reinterpret_cast<T*>(a.o) + rh * a.hd + d, v, L);
  }
}

struct SharedPlan {
  int whole, tr, NT, RT, NPc, NSc, NP, pchunk, schunk;
  int64_t units, own_blocks;
};

// Waves of the whole form's workgroup: past 64 dimensions a wave's registers and LDS leave room for four.
int whole_waves(int64_t hd) { return hd <= 64 ? 8 : 4; }
// Keys of one block of a walk (Walk::KB).
int block_keys(int64_t hd, int dtype) {
  return dtype == ESGPT_BF16 ? (hd <= 64 ? Walk<bf16, 2>::KB : Walk<bf16, 4>::KB)
                             : (hd <= 64 ? Walk<float, 2>::KB : Walk<float, 4>::KB);
}

// Whole or split, and how finely. The whole form saves the second launch and the parts' traffic but runs 16 rows a
// workgroup and one workgroup of eight waves (above 64 dimensions two of four) a CU at a time; its rounds cost what its
// busiest wave's chain of blocks costs (steps: those of the history and those of its trajectories' own rows). A tile is
// 16 rows, or 8 or 4 while there are fewer workgroups than CUs: the history is then read by more of them, out of L2,
// and each has fewer trajectories (32x16 256+64 h4: 16 rows 13.8, 8 rows 11.8). Measured in graph replays, whole / split
// us (groups x trajectories, history + own rows, heads; hd 64 bf16 if not said):
//   the busiest wave's chain of blocks is short: one; two in bf16 if half the waves have no history; up to 32 dimensions
//     one more, three in bf16. In a graph 8x4 100+10 h4 7.1 / 8.4; 1x4 40+6 h4 f32 hd16 6.4 / 7.2; 4x4 100+100 h4 9.0 /
//     9.5; 8x30 3+5 h1 hd128 8.7 / 8.9. At the rule's end a replayed call loses, 4x16 500+60 h4 hd32 8.2 / 8.0; 4x8 200+20
//     h4 f32 hd16 8.1 / 7.7; 2x13 106+189 h5 hd16 8.7 / 7.9; 5x2 691+109 h8 hd16 8.8 / 7.7; 3x5 900+50 h4 hd16 9.1 / 7.8,
//     and an eager one, which pays 3 us of host time for the second launch and its workspace, gains more: 8.5 / 11.4, 8.2 /
//     11.4, 9.1 / 11.8, 9.1 / 11.6, 9.5 / 11.5. Longer chains lose: 8x8 400+40 h4 10.0 / 9.0, 1x8 600+30 h8 10.4 / 8.8,
//     16x4 87+288 h2 hd24 10.8 / 7.8, 8x4 300+30 h4 hd128 12.3 / 9.9, f32 4x16 256+64 h4 13.3 / 11.3, f32 2x13 106+189 h5
//     hd16 12.2 / 8.0
//   smaller tiles for half the CUs or more, and a chain of at most three: 32x16 256+64 h4 11.8 / 15.2; 32x8 256+64 h4
//     9.3 / 11.7; 16x16 256+64 h4 f32 14.1 / 15.3 (a longer history: 4x16 1000+20 h8 13.3 / 10.4, 4x64 2048+32 h8 18.8 /
//     17.4)
//   16-row tiles for every CU: by an estimate of both in us. Whole: 8 + 2.8 (f32 3.2) a step and round. Split: 14 + 1.2
//     (f32 1.6) a step and workgroup of a CU, 32 rows a tile 1.6 (2.6), + 0.002 a block of own rows; all by a block's
//     bytes / 16 KB.
//     One full round, or short histories: 32x8 512+24 window 32 h8 9.0 / 15.2; 32x16 1000+20 h8 21.3 / 25.3, f32 36.9 /
//       38.6; 32x16 512+128 h8 f32 55.1 / 62.6; 32x128 256+64 h4 63.8 / 76.8; 32x64 256+20 h4 hd128 27.2 / 41.1, f32 46.5 /
//       67.5; f32 hd128 16x64 1000+20 h8 79.9 / 99.3, 64x16 256+64 h8 103 / 119
//     A round begun for a few workgroups: 33x8 1500+20 h8 37.5 / 29.7; 20x32 2000+20 h8 44.3 / 31.8; 24x40 2000+20 h8
//       f32 hd128 191 / 172. Many row tiles over a long history: 8x64 two events 4096+20 h8 54.6 / 39.4, 32x40 two
//       3000+20 h8 119 / 89.6
//     One wave's chain of own rows: 64x1 512+400 h8 38.6 / 27.1, 64x2 41.7 / 35.8
// Without a history the split form's waves are the whole of it, and write directly where one chunk holds a trajectory.
// The split form's chunks aim at one workgroup per CU: 256 / 512 units 8x32 16384+64 h8 57.4 / 59.4, 8x8 8192+32 h8 f32
// 51.3 / 53.9, 16x4 1024+33 h4 f32 16.5 / 17.2, 24x40 2000+20 h8 47.5 / 53.1 (more parts cost more joins); own rows at
// 1,024 waves: 16x16 256+64 f32 15.7 against 19.7 at 4,096. In f32 up to 32 dimensions a workgroup has little in
// flight, and two a CU pay: 8x32 8192+32 h8 hd32 45.5 -> 38.4, 2x64 4096+32 h8 hd16 17.0 -> 14.9 (bf16 19.3 -> 20.6,
// 10.7 -> 10.6).
// History tiles of 32 rows halve the reads but leave half the workgroups to share a history; they pay where each wave
// still has 256 keys. 16 / 32 rows: 24x40 2000+20 h8 53.1 / 47.2, 20x32 2000 33.9 / 31.9, 4x32 16384 h8 f32 79.4 /
// 65.2, 16x32 4096 f32 83.9 / 71.2; fewer: 4x20 1000 h4 9.5 / 11.1, 1x40 6000 h8 14.0 / 15.1, 8x32 2048 f32 29.0 /
// 27.7. At 128 dimensions (f32: above 64) two accumulators leave one wave a SIMD: 24x40 2000 h8 77.3 / 96.4, 1x40 6000
// 18.5 / 25.7.
SharedPlan shared_plan(int64_t G, int64_t S, int64_t Lq, int64_t H, int64_t hd, int64_t prefix_cap, int64_t cap,
                       int64_t window, int dtype) {
  SharedPlan p{};
  constexpr int64_t kCus = 256;
  const bool bf = dtype == ESGPT_BF16;
  const int64_t M = (S / G) * Lq, kb = block_keys(hd, dtype), nw = whole_waves(hd);
  const int64_t pspan = window ? std::min(prefix_cap, window + 16) : prefix_cap;
  const int64_t sspan = window ? std::min(cap, window + Lq + 16) : cap;
  // split
  const int64_t round = kWaves * kb, want = !bf && hd <= 32 ? 2 * kCus : kCus;
  p.NT = M > 16 && hd <= (bf ? 96 : 64) && G * H * cdiv(M, 32) * pspan >= 256 * kWaves * want ? 2 : 1;
  p.RT = (int)cdiv(M, 16 * p.NT);
  const int64_t base = G * H * p.RT;
  p.NPc = pspan ? (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(want, base), cdiv(pspan, round), 48})) : 0;
  p.pchunk = p.NPc ? (int)(cdiv(cdiv(pspan, p.NPc), round) * round) : 0;
  p.NPc = p.NPc ? (int)cdiv(pspan, p.pchunk) : 0;
  p.NSc = (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(4 * kCus, S * H), cdiv(sspan, 2 * kb), 16}));
  p.schunk = (int)(cdiv(cdiv(sspan, p.NSc), kb) * kb);
  p.NSc = (int)cdiv(sspan, p.schunk);
  p.NP = p.NPc + p.NSc;
  p.units = base * p.NPc;
  p.own_blocks = cdiv(S * H * p.NSc, kWaves);
  // whole
  int64_t tr = 16;
  while (tr > 4 && G * H * cdiv(M, tr) < kCus) tr /= 2;
  const int64_t seqs = std::min<int64_t>(cdiv(std::min<int64_t>(M, tr), Lq) + (Lq > 1), S / G);  // of a tile
  const int64_t steps = cdiv(pspan, nw * kb), own_steps = cdiv(seqs, nw) * cdiv(sspan, kb), units = G * H * cdiv(M, tr);
  const double block = (double)(cdiv(hd, 32) * 32 * kb * 2 * (bf ? 2 : 4)) / 16384;
  const double whole_us = 8 + (bf ? 2.8 : 3.2) * block * nw / 8 * cdiv(units, kCus) * (steps + own_steps);
  const double a_cu = 0.5 * std::max<int64_t>(2, cdiv(2 * p.units, kCus));  // workgroups
  const double split_us = 14 + block * ((p.NT == 2 ? (bf ? 1.6 : 2.6) : (bf ? 1.2 : 1.6)) * a_cu * (p.pchunk / round) +
                                        0.002 * (double)(S * H) * cdiv(sspan, kb));
  const int64_t hist = cdiv(pspan, kb);
  int64_t chain = 0;
  for (int64_t w = 0; w < nw; ++w)
    chain = std::max(chain, cdiv(std::max<int64_t>(hist - w, 0), nw) +
                                cdiv(std::max<int64_t>(seqs - (nw - 1 - w), 0), nw) * cdiv(sspan, kb));
  p.whole = pspan > 0 && (chain <= 1 + (hd <= 32) + (bf && (hd <= 32 || 2 * hist <= nw)) ||
                          (tr == 16 && units >= kCus && whole_us <= split_us) ||
                          (units >= kCus / 2 && steps <= 1 && own_steps <= 2));
  if (p.whole) {
    p.tr = (int)tr;
    p.RT = (int)cdiv(M, tr);
    p.units = units;
    p.NT = p.NP = 1;
    p.NPc = p.NSc = p.pchunk = p.schunk = 0;
    p.own_blocks = 0;
  }
  return p;
}

template <typename T>
int launch_shared(const SharedPlan& p, const SharedArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(p.units + p.own_blocks)), block(64 * kWaves);
  const int kd = (a.hd + 31) / 32;
  if (p.whole) {
    const dim3 wide(64 * whole_waves(a.hd));
    if (kd == 1) shared_whole_kernel<T, 1, 8><<<grid, wide, 0, st>>>(a);
    else if (kd == 2) shared_whole_kernel<T, 2, 8><<<grid, wide, 0, st>>>(a);
    else if (kd == 3) shared_whole_kernel<T, 3, 4><<<grid, wide, 0, st>>>(a);
    else shared_whole_kernel<T, 4, 4><<<grid, wide, 0, st>>>(a);
    ESGPT_LAUNCH_CHECK();
    return ESGPT_OK;
  }
#define SHARED(KD)                                                                        \
  do {                                                                                    \
    if constexpr (KD <= (sizeof(T) == 2 ? 3 : 2)) {                                       \
      if (p.NT == 2) {                                                                    \
        shared_kernel<T, KD, 2><<<grid, block, 0, st>>>(a);                               \
        break;                                                                            \
      }                                                                                   \
    }                                                                                     \
    shared_kernel<T, KD, 1><<<grid, block, 0, st>>>(a);                                   \
  } while (0)
  if (kd == 1) SHARED(1);
  else if (kd == 2) SHARED(2);
  else if (kd == 3) SHARED(3);
  else SHARED(4);
#undef SHARED
  ESGPT_LAUNCH_CHECK();
  if (p.NP > 1) {
    int width = 1;
    while (4 * width < a.hd) width *= 2;
    const int64_t rows = (int64_t)a.S * a.Lq * a.H;
    shared_join_kernel<T><<<(unsigned)cdiv(rows, 4), 256, 0, st>>>(a, rows, width);
    ESGPT_LAUNCH_CHECK();
  }
  return ESGPT_OK;
}

// 0 for a window that no distance within the caps leaves.
int64_t cut_window(int64_t window, int64_t prefix_cap, int64_t cap) { return window < prefix_cap + cap ? window : 0; }

bool shared_ok(int64_t G, int64_t S, int64_t Lq, int64_t H, int64_t hd, int64_t prefix_cap, int64_t cap, int64_t window,
               int dtype) {
  return G > 0 && S >= G && S % G == 0 && Lq >= 1 && Lq <= kMaxLq && H > 0 && hd > 0 && hd <= 128 &&
         hd % (dtype == ESGPT_BF16 ? 8 : 4) == 0 && (dtype == ESGPT_F32 || dtype == ESGPT_BF16) && prefix_cap >= 0 &&
         cap >= 1 && prefix_cap <= (int64_t)1 << 29 && cap <= (int64_t)1 << 29 && window >= 0 &&
         S * Lq * H < (int64_t)1 << 28;
}

}  // namespace

extern "C" {

size_t esgpt_attn_decode_shared_workspace(int64_t G, int64_t S, int64_t Lq, int64_t H, int64_t hd, int64_t prefix_cap,
                                          int64_t cap, int64_t window, int dtype) {
  if (!shared_ok(G, S, Lq, H, hd, prefix_cap, cap, window, dtype)) return 0;
  const SharedPlan p = shared_plan(G, S, Lq, H, hd, prefix_cap, cap, cut_window(window, prefix_cap, cap), dtype);
  return p.NP > 1 ? (size_t)(S * Lq * H * p.NP) * (2 + hd) * sizeof(float) : 0;
}

int esgpt_attn_decode_shared(const void* q, const void* k_pages, const void* v_pages, int64_t n_pages,
                             int64_t page_size, const int32_t* prefix_table, int64_t prefix_w,
                             const int32_t* prefix_lens, int64_t G, const int32_t* page_table, int64_t table_w,
                             const int32_t* past, const uint8_t* row_mask, void* o, int64_t S, int64_t Lq, int64_t H,
                             int64_t hd, int64_t prefix_cap, int64_t cap, int64_t window, int dtype, void* workspace,
                             size_t workspace_bytes, int32_t* err, void* stream) {
  if (S == 0 && Lq >= 0 && Lq <= kMaxLq) return ESGPT_OK;
  ESGPT_REQUIRE(shared_ok(G, S, Lq, H, hd, prefix_cap, cap, window, dtype));
  ESGPT_REQUIRE(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0 && n_pages >= 0 &&
                n_pages < (int64_t)1 << 31 && table_w >= 0 && table_w < (int64_t)1 << 31 && prefix_w >= 0 &&
                prefix_w < (int64_t)1 << 31 && cap <= table_w * page_size && prefix_cap <= prefix_w * page_size);
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  ESGPT_REQUIRE(q && o && past && page_table && aligned(q) && aligned(o) && (prefix_cap == 0 || (prefix_table && prefix_lens)));
  ESGPT_REQUIRE(n_pages == 0 || (k_pages && v_pages && aligned(k_pages) && aligned(v_pages)));
  const uint32_t far = window ? (uint32_t)std::min<int64_t>(window, ~0u) : ~0u;
  window = cut_window(window, prefix_cap, cap);
  const SharedPlan p = shared_plan(G, S, Lq, H, hd, prefix_cap, cap, window, dtype);
  // a launch holds fewer than 2^32 threads
  constexpr int64_t kThreads = ((int64_t)1 << 32) - 1;
  ESGPT_REQUIRE((p.units + p.own_blocks) * 64 * (p.whole ? whole_waves(hd) : kWaves) <= kThreads &&
                cdiv(S * Lq * H, 4) * 256 <= kThreads);
  SharedArgs a{};
  if (p.NP > 1) {
    const size_t rows = (size_t)(S * Lq * H * p.NP);
    ESGPT_REQUIRE(workspace && aligned(workspace) && workspace_bytes >= rows * (2 + hd) * sizeof(float));
    a.po = reinterpret_cast<float*>(workspace);
    a.ml = a.po + rows * hd;
  }
  a.q = q;
  a.kp = k_pages;
  a.vp = v_pages;
  a.o = o;
  a.prefix_table = prefix_table;
  a.prefix_lens = prefix_lens;
  a.table = page_table;
  a.past = past;
  a.row_mask = row_mask;
  a.err = err;
  a.n_pages = n_pages;
  a.prefix_w = prefix_w;
  a.table_w = table_w;
  a.S = (int)S;
  a.n = (int)(S / G);
  a.Lq = (int)Lq;
  a.H = (int)H;
  a.hd = (int)hd;
  a.psl = 0;
  while ((1 << a.psl) < page_size) ++a.psl;
  a.prefix_cap = (int)prefix_cap;
  a.cap = (int)cap;
  a.window = (int)window;
  a.owin = window < cap ? (int)window : 0;
  a.far = far;
  a.M = (int)((S / G) * Lq);
  a.RT = p.RT;
  a.tr = p.tr;
  a.NPc = p.NPc;
  a.NSc = p.NSc;
  a.NP = p.NP;
  a.pchunk = p.pchunk;
  a.schunk = p.schunk;
  a.units = (int)p.units;
  if (dtype == ESGPT_F32) return launch_shared<float>(p, a, as_stream(stream));
  return launch_shared<bf16>(p, a, as_stream(stream));
}

}  // extern "C"
