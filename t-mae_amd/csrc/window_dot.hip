// Scaled-dot-product attention inside 8x8 windows of the token grid.
//
//   P_ij = softmax_j(scale q_i . k_j) over the keys j of the query's window,  o_i = sum_j P_ij v_j;  a window without keys: o_i = 0
//   backward, P recomputed from q and k (nothing is kept of the forward but its inputs: a log-sum-exp a row and head, 4 bytes at a time in
//   rows that lie apart, took longer to write and read than the row maxima and sums take to compute again):
//   dV_j = sum_i P_ij dO_i,  dP_ij = dO_i . v_j,  dS_ij = scale P_ij (dP_ij - sum_j P_ij dP_ij),  dQ_i = sum_j dS_ij k_j,  dK_j = sum_i dS_ij q_i
//
// Tiles of 16 tokens.  A logit tile is computed with the keys as its rows and the queries as its columns: the accumulators' layout --
// lane (g, i) = (lane >> 4, lane & 15) holds rows 4g .. 4g+3 of column i -- is also what the next product takes as its B operand, row
// 4g + r in step r, so that the probabilities go into it without leaving the registers (float32 whole, bfloat16 as the sum of two).
//
// Bound: HBM, at 14 to 24 FLOPs a byte; but rows lie apart and windows are small, so what costs is getting rows in and out.  The lanes of an
// operand stand in 16 rows: read straight into that layout, an instruction touches a line for every few lanes.  Rows therefore travel in
// 16-byte pieces, whole pieces of a line by neighbouring lanes, through LDS images; all of a window's rows are requested at once.  Padding
// rows to tiles is what the matrix unit pays for; three sizes of windows (up to 16, 32 and 64 tokens) keep it small.  Eight frames at stage 1
// (375 k tokens, 8 heads of 16, bfloat16): forward 104 us, backward 187 us, 4.2 and 3.9 TB/s of counted HBM traffic (110 and 223 us with a
// profiler's trace around every launch; the comparisons below are of traced launches).
//
// A slot behind a window's last token stands for its first one: it is read, its probability is set to 0 (and V and dO are zeros there,
// which an infinity next to them needs), and nothing is stored for it.
#include "common.h"
#include <type_traits>

namespace {

constexpr int WIN = 8;
constexpr int WL_HDR = 8;                  // the work list: tmae_window_worklist
constexpr float LOG2E = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct DotArgs {
  const void *q, *k, *v, *g;               // g: dO
  unsigned pq, pk, pv, pg;                 // row pitches in bytes
  void *o, *dq, *dk, *dv;
  unsigned po, pdq, pdk, pdv;
  const int32_t *grid_q, *grid_k, *wl;
  int64_t mq, mk, nwin;
  int nhead, batch, ny, nx, Wy, Wx, s;
  float scale;
};

// row `token` of a tensor: one multiply-add of 32 x 32 bits onto 64, where a pitch of 64 bits takes three of them
__device__ __forceinline__ char* row_of(const void* base, int token, unsigned pitch) {
  return (char*)base + (unsigned long long)(unsigned)token * pitch;
}

// LDS operations of a wave execute in order: this keeps the compiler to the order they are written in.  In bfloat16 every wave works in
// images of its own; the waves of a workgroup meet where they move rows for each other.
__device__ __forceinline__ void order_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A barrier of the workgroup for what is in LDS alone: rows on their way from or to memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The windows of a launch: those of the work list's classes `from`, `from` - 1, ... `to` one after the other (larger windows first), or
// every window of the grids where there is no list.  A wave takes every step-th one.  The list's entry, the cells and the rows are three
// loads that wait for each other: a wave reads 64 of its entries at once (a lane each), and requests the cells of the next window before
// it works on the present one.  No load stands behind a branch -- it would be waited for there -- so places that do not exist are
// replaced by ones that do.
struct Walk {
  int n, e, step, from, to;                // windows in all, the present one
  int entries, at;                         // this lane's entry of the 64, the next window's among them
  int tq, tk;                              // this lane's cell of the present window: row numbers, -1 where it is empty
  int nq, nk;                              // ... of the next one, if it is a cell of the grid
  bool nin;

  __device__ __forceinline__ static int count(const DotArgs& a, int cls) {
    const int c = a.wl[cls];
    return c < 0 ? 0 : c < (int)a.nwin ? c : (int)a.nwin;
  }
  __device__ __forceinline__ void read_entries(const DotArgs& a, int first) {
    int x = first + (int)(threadIdx.x & 63) * step;
    if (x >= n || x < first) x = n - 1;
    entries = x;
    at = 0;
    if (a.wl) {
      int cls = from;
      for (int c = from; c > to; --c) {
        const int k = count(a, c);
        if (cls == c && x >= k) { x -= k; cls = c - 1; }
      }
      entries = a.wl[WL_HDR + cls * a.nwin + x];
      asm volatile("" : "+v"(entries));      // waited for here, once in 64 windows, and not where the two ways meet again
    }
  }
  __device__ __forceinline__ void request_cells(const DotArgs& a) {
    const int lane = threadIdx.x & 63, u = __builtin_amdgcn_readlane(entries, at);
    int b, wcy, wcx;
    if (a.wl) {
      b = u >> 16; wcx = (u >> 8) & 255; wcy = u & 255;
    } else {
      wcy = u % a.Wy; wcx = u / a.Wy % a.Wx; b = u / (a.Wy * a.Wx);
    }
    const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
    const bool in = b >= 0 && b < a.batch && y >= 0 && y < a.ny && x >= 0 && x < a.nx;
    int cell = in ? (b * a.ny + y) * a.nx + x : 0;                   // batch * ny * nx < 2^31
    asm volatile("" : "+v"(cell));           // (the loads stay outside of the condition)
    nq = a.grid_q[cell];
    nk = a.grid_k[cell];
    nin = in;
  }
  __device__ __forceinline__ Walk(const DotArgs& a, int from_, int to_, int first, int step_) : e(first - step_), step(step_), from(from_), to(to_) {
    n = (int)a.nwin;
    if (a.wl) {
      n = 0;
      for (int c = from; c >= to; --c) n += count(a, c);
    }
    tq = tk = nq = nk = -1;
    nin = false;
    if (first < n) {
      read_entries(a, first);
      request_cells(a);
    }
  }
  __device__ __forceinline__ bool next(const DotArgs& a) {
    if (e >= n - step) return false;
    e += step;
    tq = nin && nq < a.mq ? nq : -1;       // a row number outside the tensors counts as an empty cell
    tk = nin && nk < a.mk ? nk : -1;
    if (++at == 64) read_entries(a, e < n - step ? e + step : e);
    request_cells(a);                      // (behind the last window: once more some window of the list)
    return true;
  }
  // the tokens in cell order into toks[0] (queries) and toks[1] (keys), at most `most` of each; the slots behind repeat the first one
  __device__ __forceinline__ void tokens(int (*toks)[64], int most, int& Tq, int& Tk) const {
    const int lane = threadIdx.x & 63;
    const unsigned long long q = __ballot(tq >= 0), k = __ballot(tk >= 0), below = (1ull << lane) - 1ull;
    Tq = min(__popcll(q), most);
    Tk = min(__popcll(k), most);
    const int fq = __builtin_amdgcn_readlane(tq, q ? __ffsll(q) - 1 : 0), fk = __builtin_amdgcn_readlane(tk, k ? __ffsll(k) - 1 : 0);
    // every lane writes one slot of each list: the tokens' ranks first, then the others the slots behind (a full list has none)
    const int rq = __popcll(q & below), rk = __popcll(k & below), sq = __popcll(q), sk = __popcll(k);
    order_lds();
    toks[0][tq >= 0 ? rq : sq + lane - rq] = tq >= 0 ? tq : fq;
    toks[1][tk >= 0 ? rk : sk + lane - rk] = tk >= 0 ? tk : fk;
    order_lds();
  }
};

// ------------------------------------------------------------------------------------------------------------------- float32
// Four waves of a workgroup share the windows of up to 16 NT tokens: NT of them the tiles of one head, 4 / NT heads at a time -- 64 rows
// of each tensor in LDS whatever the window's size.  A wave takes one tile of queries (out, dQ and the rows' maxima, sums and sum_j P dP),
// then, in the backward, one tile of keys (dK, dV).  Operands come from LDS: pieces of rows for the products over the channels, single
// values of four rows for those over the tokens.  One frame of stage 2 (16 k tokens, 8 heads of 32): forward 21 us, backward 47 us; a wave
// for a whole (window, head), its rows read straight into the operands' layout, took 125 us for both.
__device__ __forceinline__ float lanes4_sum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float lanes4_max(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }

template <int DH> struct Rows32 {
  static constexpr int PITCH = DH + 4, KD = DH / 4, CT = DH / 16, IMAGE = 64 * PITCH;      // floats
  struct Piece { f32x4 v[KD / 4]; };         // of row i: channels 4g .. 4g + 3 of every 16
  static __device__ __forceinline__ Piece piece(const float* tile, int g, int i) {
    Piece p;
#pragma unroll
    for (int j = 0; j < KD / 4; ++j) p.v[j] = *reinterpret_cast<const f32x4*>(tile + i * PITCH + 16 * j + 4 * g);
    return p;
  }
  static __device__ __forceinline__ f32x4 over_channels(const Piece& a, const Piece& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KD / 4; ++j)
#pragma unroll
      for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j][s], b.v[j][s], c, 0, 0, 0);
    return c;
  }
  // c[ct] += channels 16 ct .. + 15 of the tile's rows (as rows of the result) x b (columns), over the tile's 16 tokens
  static __device__ __forceinline__ void over_tokens(const float* tile, const f32x4& b, f32x4* c, int g, int i) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) c[ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile[(4 * g + r) * PITCH + 16 * ct + i], b[r], c[ct], 0, 0, 0);
  }
  static __device__ __forceinline__ void store(float* row, int g, const f32x4* v, float by) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<f32x4*>(row + 16 * ct + 4 * g) = v[ct] * by;
  }
};

template <int DH, int NT, bool BWD> __device__ __forceinline__ void f32_role(const DotArgs& a, int first, int step, int group, int (*toks)[64], float* lds) {
  using R = Rows32<DH>;
  constexpr int CT = R::CT, ROWS = NT * 16, HPB = 4 / NT, NI = BWD ? 4 : 3;
  constexpr int LPR = DH / 4, RP = 256 / LPR, PASSES = 64 / RP, TILE = 16 * R::PITCH;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
  const int t = w % NT, hh = w / NT, head = group * HPB + hh;
  float *top = lds + NI * R::IMAGE, *inv = top + 64, *dot = inv + 64;           // per row: c * the largest logit, 1 / sum_j, sum_j P dP
  const float c = a.scale * LOG2E;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  for (Walk walk(a, NT == 4 ? 3 : NT == 2 ? 2 : 1, NT == 4 ? 3 : NT == 2 ? 2 : 0, first, step); walk.next(a);) {
    int Tq, Tk;
    walk.tokens(toks, ROWS, Tq, Tk);
    if (Tq == 0 || Tk == 0) {
      if (t == 0 && head < a.nhead) {
        const int at = (head * DH + lane % LPR * 4) * 4;
        for (int r = lane / LPR; r < Tq; r += 64 / LPR)
          *reinterpret_cast<f32x4*>(row_of(BWD ? a.dq : a.o, toks[0][r], BWD ? a.pdq : a.po) + at) = zero;
        if (BWD)
          for (int r = lane / LPR; r < Tk; r += 64 / LPR) {
            *reinterpret_cast<f32x4*>(row_of(a.dk, toks[1][r], a.pdk) + at) = zero;
            *reinterpret_cast<f32x4*>(row_of(a.dv, toks[1][r], a.pdv) + at) = zero;
          }
      }
      continue;
    }
    f32x4 rows[NI][PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int row = p * RP + (int)threadIdx.x / LPR, slot = row % ROWS;
      int h = group * HPB + row / ROWS;
      if (h >= a.nhead) h = a.nhead - 1;
      const int tq = toks[0][slot], tk = toks[1][slot], col = (h * DH + (int)threadIdx.x % LPR * 4) * 4;
      rows[0][p] = *reinterpret_cast<const f32x4*>(row_of(a.k, tk, a.pk) + col);
      rows[1][p] = *reinterpret_cast<const f32x4*>(row_of(a.v, tk, a.pv) + col);
      rows[2][p] = *reinterpret_cast<const f32x4*>(row_of(a.q, tq, a.pq) + col);
      if constexpr (BWD) rows[3][p] = *reinterpret_cast<const f32x4*>(row_of(a.g, tq, a.pg) + col);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {       // slots without a token hold zeros: 0 times a probability of 0, whatever the tokens hold
      const int slot = (p * RP + (int)threadIdx.x / LPR) % ROWS;
      if (slot >= Tk) rows[0][p] = rows[1][p] = zero;
      if (slot >= Tq) { rows[2][p] = zero; if constexpr (BWD) rows[3][p] = zero; }
    }
    lds_barrier();                         // the window before is done with
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int n = 0; n < NI; ++n)
        *reinterpret_cast<f32x4*>(lds + n * R::IMAGE + (p * RP + (int)threadIdx.x / LPR) * R::PITCH + (int)threadIdx.x % LPR * 4) = rows[n][p];
    lds_barrier();
    const int nq = (Tq + 15) >> 4, nk = (Tk + 15) >> 4;
    const float *K = lds + hh * ROWS * R::PITCH, *V = K + R::IMAGE, *Q = K + 2 * R::IMAGE, *G = K + 3 * R::IMAGE;
    const bool mine = head < a.nhead;
    if (mine && t < nq) {
      const typename R::Piece qf = R::piece(Q + t * TILE, g, i);
      typename R::Piece gf;
      if constexpr (BWD) gf = R::piece(G + t * TILE, g, i);
      f32x4 p[NT], dp[NT];
      float mx = -INFINITY, l = 0.f, d = 0.f;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        if (kt < nk) {
          p[kt] = R::over_channels(R::piece(K + kt * TILE, g, i), qf);              // rows = keys, column = query i
          if constexpr (BWD) dp[kt] = R::over_channels(R::piece(V + kt * TILE, g, i), gf);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (kt * 16 + 4 * g + r >= Tk) p[kt][r] = -INFINITY;
            mx = fmaxf(mx, p[kt][r]);
          }
        }
      }
      mx = lanes4_max(mx) * c;
      f32x4 o[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] = zero;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        if (kt < nk) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[kt][r] = __builtin_amdgcn_exp2f(fmaf(p[kt][r], c, -mx));
            l += p[kt][r];
            if constexpr (BWD) d += p[kt][r] * dp[kt][r];
          }
          if constexpr (!BWD) R::over_tokens(V + kt * TILE, p[kt], o, g, i);        // rows = channels, column = query i
        }
      }
      const float il = 1.f / lanes4_sum(l);
      const int tq = toks[0][t * 16 + i];
      if constexpr (BWD) {
        d = lanes4_sum(d) * il;
        const int row = hh * ROWS + t * 16 + i;
        if (g == 0) { top[row] = mx; inv[row] = t * 16 + i < Tq ? il : 0.f; dot[row] = d; }          // no query: P = dS = 0
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
          if (kt < nk) {
#pragma unroll
            for (int r = 0; r < 4; ++r) p[kt][r] = p[kt][r] * il * (dp[kt][r] - d);
            R::over_tokens(K + kt * TILE, p[kt], o, g, i);
          }
        }
        if (t * 16 + i < Tq) R::store((float*)row_of(a.dq, tq, a.pdq) + head * DH, g, o, a.scale);
      } else {
        if (t * 16 + i < Tq) R::store((float*)row_of(a.o, tq, a.po) + head * DH, g, o, il);
      }
    }
    if constexpr (BWD) {
      lds_barrier();
      if (mine && t < nk) {
        const typename R::Piece kf = R::piece(K + t * TILE, g, i), vf = R::piece(V + t * TILE, g, i);
        f32x4 dk[CT], dv[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) dk[ct] = dv[ct] = zero;
        for (int qt = 0; qt < nq; ++qt) {
          f32x4 p = R::over_channels(R::piece(Q + qt * TILE, g, i), kf), ds = R::over_channels(R::piece(G + qt * TILE, g, i), vf);
          const int row = hh * ROWS + qt * 16 + 4 * g;                              // rows = queries, column = key i
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool present = inv[row + r] != 0.f;
            p[r] = present ? __builtin_amdgcn_exp2f(fmaf(p[r], c, -top[row + r])) * inv[row + r] : 0.f;
            ds[r] = present ? p[r] * (ds[r] - dot[row + r]) : 0.f;
          }
          R::over_tokens(G + qt * TILE, p, dv, g, i);
          R::over_tokens(Q + qt * TILE, ds, dk, g, i);
        }
        if (t * 16 + i < Tk) {
          const int tk = toks[1][t * 16 + i];
          R::store((float*)row_of(a.dk, tk, a.pdk) + head * DH, g, dk, a.scale);
          R::store((float*)row_of(a.dv, tk, a.pdv) + head * DH, g, dv, 1.f);
        }
      }
    }
  }
}

struct Roles32 { int n4, n2, n1, h4, h2, h1; };      // workgroups along the windows of each size, and along the heads
// Three workgroups a CU in the backward (10 registers of heads of 32 spilled: 59 us a frame of 16 k tokens, 67 with room for two and none spilled)
template <int DH, bool BWD>
__global__ __launch_bounds__(256, (BWD && DH == 64 ? 2 : 3)) void dot_f32_kernel(DotArgs a, Roles32 n) {
  extern __shared__ __attribute__((aligned(16))) float lds32[];
  __shared__ int toks_[4][2][64];
  int (*toks)[64] = toks_[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
  int u = blockIdx.x;
  if (u < n.n4 * n.h4) { f32_role<DH, 4, BWD>(a, u / n.h4, n.n4, u % n.h4, toks, lds32); return; }
  u -= n.n4 * n.h4;
  if (u < n.n2 * n.h2) { f32_role<DH, 2, BWD>(a, u / n.h2, n.n2, u % n.h2, toks, lds32); return; }
  u -= n.n2 * n.h2;
  f32_role<DH, 1, BWD>(a, u / n.h1, n.n1, u % n.h1, toks, lds32);
}

// The windows that are in no list: zero rows for queries without a key (out, or dq) and for keys without a query (dk, dv).  A wave per
// window, a lane per cell, whole rows at a time.
struct Orphans { char *q; int64_t ldq; char *k, *v; int64_t ldk, ldv; int row16; };        // pitches in bytes, 16-byte pieces of a row
__device__ __forceinline__ void orphan_role(const DotArgs& a, const Orphans& z, int64_t first, int64_t step) {
  const int lane = threadIdx.x & 63;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t u = first; u < a.nwin; u += step) {
    const int e = (int)u, wcy = e % a.Wy, wcx = e / a.Wy % a.Wx, b = e / (a.Wy * a.Wx);
    const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
    const bool in = y >= 0 && y < a.ny && x >= 0 && x < a.nx;
    const int cell = in ? (b * a.ny + y) * a.nx + x : 0;
    int tq = a.grid_q[cell], tk = a.grid_k[cell];
    if (!in || tq >= a.mq) tq = -1;
    if (!in || tk >= a.mk) tk = -1;
    const unsigned long long q = __ballot(tq >= 0), k = __ballot(tk >= 0);
    if (z.q && !k)
      for (unsigned long long m = q; m; m &= m - 1) {
        uint4* r = reinterpret_cast<uint4*>(z.q + (int64_t)__builtin_amdgcn_readlane(tq, __ffsll(m) - 1) * z.ldq);
        for (int c = lane; c < z.row16; c += 64) r[c] = zero;
      }
    if (z.k && !q)
      for (unsigned long long m = k; m; m &= m - 1) {
        const int64_t t = __builtin_amdgcn_readlane(tk, __ffsll(m) - 1);
        uint4 *r = reinterpret_cast<uint4*>(z.k + t * z.ldk), *v = reinterpret_cast<uint4*>(z.v + t * z.ldv);
        for (int c = lane; c < z.row16; c += 64) { r[c] = zero; v[c] = zero; }
      }
  }
}
__global__ __launch_bounds__(256) void dot_orphan_kernel(DotArgs a, Orphans z) {
  orphan_role(a, z, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), (int64_t)gridDim.x * 4);
}

// ------------------------------------------------------------------------------------------------------------------ bfloat16
// The same products on the bfloat16 matrix instructions.  Their operands want the 16 rows of a tile in 16 neighbouring lanes: loaded that
// way straight from the tensors, each instruction touches 16 lines per 16 lanes, and the first kernels waited for that.  So rows travel in
// 16-byte chunks, neighbouring lanes on neighbouring chunks, into row images in LDS, and the operands are read there: pieces of a row for
// the products over the channels (logits, dP), columns (ds_read_b64_tr_b16 returns four rows of one column) for the products over tokens.
// Results go back the same way: into the image, and out in whole rows.
//
// P and dS enter their products as the sum of two bfloat16 each (2^-15 of a probability, 2^-16 of dS; sums, maxima and everything else stay
// float32): the results' error is that of their own rounding.  Rounded to one bfloat16 they would add as much again (2-norms: 0.0024 of the
// gradients, not 0.0017) and save 35 of 220 us of the backward at stage 1, 6 of 85 across frames of stage 2.

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int TILE_PITCH = 40, TILE_BYTES = 16 * TILE_PITCH;             // a 16x16 bfloat16 tile in LDS

__device__ __forceinline__ unsigned pack2(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ s16x4 pack4(const f32x4& v) { return __builtin_bit_cast(s16x4, u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])}); }
__device__ __forceinline__ s16x4 read_columns(const char* lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)lds);
}
// sum / maximum over the 4 lanes that share a column, in every one of them.  The sum is a product with ones: the matrix unit has time,
// the vector unit does not.  The maximum is the median with infinity, which asks for no quieting of a NaN first (a NaN lost here is still
// in its probability).
__device__ __forceinline__ float column_sum(float v) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_f32_16x16x4f32(1.f, v, zero, 0, 0, 0)[0];
}
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = larger(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return larger(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// One head's columns of a row image, 16 rows (a tile) at a time.
template <int DH, int PITCH> struct Rows {
  static constexpr int FR = DH / 4, CT = DH / 16;
  struct Piece { unsigned u[FR / 2]; };    // of row i: channels 4g.. (DH 16), 8g.. (32), 8g.. and 32 + 8g.. (64)
  static __device__ __forceinline__ Piece piece(const char* tile, int g, int i) {
    Piece f;
    if constexpr (FR == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(tile + i * PITCH + 8 * g);
      f.u[0] = v.x; f.u[1] = v.y;
    } else {
#pragma unroll
      for (int j = 0; j < FR / 8; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(tile + i * PITCH + 64 * j + 16 * g);
        f.u[4 * j] = v.x; f.u[4 * j + 1] = v.y; f.u[4 * j + 2] = v.z; f.u[4 * j + 3] = v.w;
      }
    }
    return f;
  }
  // rows 4g .. 4g + 3 of channel 16 ct + i
  static __device__ __forceinline__ s16x4 columns(const char* tile, int g, int i, int ct) {
    return read_columns(tile + (4 * g + (i >> 2)) * PITCH + 32 * ct + 8 * (i & 3));
  }
  // the accumulators' layout: channels 16 ct + 4g .. + 3 of row i
  static __device__ __forceinline__ void put(char* tile, int g, int i, const f32x4* v) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<s16x4*>(tile + i * PITCH + 32 * ct + 8 * g) = pack4(v[ct]);
  }
  static __device__ __forceinline__ f32x4 over_channels(const Piece& a, const Piece& b, f32x4 c) {
    if constexpr (FR == 4) {
      c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < FR / 8; ++j)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, u32x4{a.u[4 * j], a.u[4 * j + 1], a.u[4 * j + 2], a.u[4 * j + 3]}),
            __builtin_bit_cast(bf16x8, u32x4{b.u[4 * j], b.u[4 * j + 1], b.u[4 * j + 2], b.u[4 * j + 3]}), c, 0, 0, 0);
    }
    return c;
  }
};
// Probabilities and their gradients on the way into the products over the tokens: as the sum of two bfloat16, 16 bits and more.  The
// instruction takes 32 tokens; where a tile has 16 the low parts ride in its second half.  Probabilities are split towards 0 and the low
// part of one above 0 stays above it (the median of the rest, the smallest normal number and the probability), so that an infinity in V or
// dO meets two positive numbers; of 0 both parts are 0.  dS is rounded to the nearest, and the rest of an infinity (a NaN, of which the median
// makes a finite number) leaves it one.
struct Split { s16x4 hi, lo; };
__device__ __forceinline__ Split probabilities(const f32x4& p) {
  u32x4 cut;
  f32x4 rest;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    cut[r] = __float_as_uint(p[r]) & 0xffff0000u;
    rest[r] = __builtin_amdgcn_fmed3f(p[r] - __uint_as_float(cut[r]), 0x1p-126f, p[r]);
  }
  return Split{__builtin_bit_cast(s16x4, u32x2{cut[0] >> 16 | cut[1], cut[2] >> 16 | cut[3]}), pack4(rest)};
}
__device__ __forceinline__ Split gradients(const f32x4& d) {
  const u32x2 h = {pack2(d[0], d[1]), pack2(d[2], d[3])};
  const f32x4 near = {__uint_as_float(h[0] << 16), __uint_as_float(h[0] & 0xffff0000u), __uint_as_float(h[1] << 16), __uint_as_float(h[1] & 0xffff0000u)};
  f32x4 rest = d - near;
#pragma unroll
  for (int r = 0; r < 4; ++r) rest[r] = __builtin_amdgcn_fmed3f(rest[r], -0x1p120f, 0x1p120f);           // finite beside an infinity
  return Split{__builtin_bit_cast(s16x4, h), pack4(rest)};
}
__device__ __forceinline__ f32x4 product32(const s16x4& a0, const s16x4& a1, const s16x4& b0, const s16x4& b1, f32x4 c) {
  const s16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// c += A B over the tokens of one tile
__device__ __forceinline__ f32x4 over_tokens(const s16x4& a, const Split& b, f32x4 c) { return product32(a, a, b.hi, b.lo, c); }
// A B over those of NK tiles (one accumulator goes through products of one shape only: a 16x16x16 right behind the 16x16x32 that it
// continues has read wrong values)
template <int NK> __device__ __forceinline__ f32x4 over_tiles(const s16x4* a, const Split* b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k + 1 < NK; k += 2) {
    c = product32(a[k], a[k + 1], b[k].hi, b[k + 1].hi, c);
    c = product32(a[k], a[k + 1], b[k].lo, b[k + 1].lo, c);
  }
  if constexpr (NK % 2 == 1) c = over_tokens(a[NK - 1], b[NK - 1], c);
  return c;
}
// a tile of them, one column a lane, into LDS and out of it with rows and columns exchanged
constexpr int WEIGHT_BYTES = 2 * TILE_BYTES;
__device__ __forceinline__ void put_tile(char* tile, int g, int i, const Split& v) {
  *reinterpret_cast<s16x4*>(tile + i * TILE_PITCH + 8 * g) = v.hi;
  *reinterpret_cast<s16x4*>(tile + TILE_BYTES + i * TILE_PITCH + 8 * g) = v.lo;
}
__device__ __forceinline__ Split turned_tile(const char* tile, int g, int i) {
  const char* at = tile + (4 * g + (i >> 2)) * TILE_PITCH + 8 * (i & 3);
  return Split{read_columns(at), read_columns(at + TILE_BYTES)};
}

// ---- windows of more than 16 tokens: a workgroup per window and four heads, a wave for each of them.  The four move the rows together,
// whole 128-byte lines at a time, and past the cache on the way out (with P and dS rounded once, backward of the large windows + the others
// in two launches, stage 1: 72 + 111 us; 74 + 119 where each wave moves its own 32 bytes of a row, 147 + 133 where those go past the cache;
// stage 2 across frames 35 + 44 and 39 + 46).  All rows of the window
// are requested at once.  Forward: K and V go through the wave's two images into registers, Q takes K's place, the output Q's.  Backward:
// K, V and Q have images; V goes into registers and dO takes its place; at the end dQ, dK and dV stand where Q, K and dO stood.
template <int DH, int NT> struct Window {
  static constexpr int PITCH = DH * 2 + 16, TILE = 16 * PITCH, IMAGE = NT * TILE;
  static constexpr int CHUNKS = DH / 8, LINE = 4 * CHUNKS, LOADS = NT * 16 * LINE / 256;      // 16-byte chunks of a head's row, of the four heads'
  using R = Rows<DH, PITCH>;
  static constexpr int CT = R::CT;

  // chunk s * 256 + threadIdx.x of the window's rows
  struct Place { int row, head, chunk; };
  static __device__ __forceinline__ Place place(int s) {
    const int q = s * 256 + (int)threadIdx.x, c = q % LINE;
    return Place{q / LINE, c / CHUNKS, c % CHUNKS};
  }
  struct Loaded { u32x4 row[LOADS]; };
  // head0: the first of the four; of heads that do not exist the last one's rows
  static __device__ __forceinline__ Loaded request(const void* base, unsigned pitch, const int* toks, int head0, int nhead) {
    Loaded l;
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
      const Place p = place(s);
      const int head = head0 + p.head < nhead ? head0 + p.head : nhead - 1;
      l.row[s] = *reinterpret_cast<const u32x4*>(row_of(base, toks[p.row], pitch) + head * DH * 2 + p.chunk * 16);
    }
    return l;
  }
  // into an image of every head (per_head bytes apart); the rows from `T` on as zeros: a probability of 0 stays one beside an infinity
  static __device__ __forceinline__ void lay(char* images, int per_head, Loaded l, int T) {
    const u32x4 none = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
      const Place p = place(s);
      *reinterpret_cast<u32x4*>(images + p.head * per_head + p.row * PITCH + p.chunk * 16) = p.row < T ? l.row[s] : none;
    }
  }
  static __device__ __forceinline__ void store(void* base, unsigned pitch, const int* toks, int T, int head0, int nhead, const char* images, int per_head) {
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
      const Place p = place(s);
      if (p.row < T && head0 + p.head < nhead)
        __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(images + p.head * per_head + p.row * PITCH + p.chunk * 16),
                                    reinterpret_cast<u32x4*>(row_of(base, toks[p.row], pitch) + (head0 + p.head) * DH * 2 + p.chunk * 16));
    }
  }
};

// NK key tiles against nq query tiles.  NK is a template parameter, so that no branch stands between a matrix instruction and its reader.
template <int DH, int NT, int NK>
__device__ __forceinline__ void fwd_window(const DotArgs& a, int Tq, int Tk, char* images, int per_head, char* A, typename Window<DH, NT>::Loaded qrows) {
  using W = Window<DH, NT>;
  using R = typename W::R;
  constexpr int CT = W::CT, TILE = W::TILE;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15, nq = (Tq + 15) >> 4;
  const char* V = A + W::IMAGE;
  typename R::Piece kf[NK];
  s16x4 vc[CT][NK];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    kf[kt] = R::piece(A + kt * TILE, g, i);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) vc[ct][kt] = R::columns(V + kt * TILE, g, i, ct);
  }
  lds_barrier();
  W::lay(images, per_head, qrows, Tq);
  lds_barrier();
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 absent;                              // of the last key tile: -inf where there is no key
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = (NK - 1) * 16 + 4 * g + r < Tk ? 0.f : -INFINITY;
  const float c = a.scale * LOG2E;
  for (int qt = 0; qt < nq; ++qt) {
    const typename R::Piece qf = R::piece(A + qt * TILE, g, i);
    f32x4 st[NK];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) st[kt] = R::over_channels(kf[kt], qf, kt == NK - 1 ? absent : zero);
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = larger(mx, st[kt][r]);
    mx = column_max(mx) * c;
    float l = 0.f;
    Split p[NK];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][r], c, -mx));
        l += st[kt][r];
      }
      p[kt] = probabilities(st[kt]);
    }
    l = column_sum(l);
    f32x4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = over_tiles<NK>(vc[ct], p);
    const float il = __builtin_amdgcn_rcpf(l);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] *= il;
    R::put(A + qt * TILE, g, i, o);
  }
}

template <int DH, int NT, int NK>
__device__ __forceinline__ void bwd_window(const DotArgs& a, int Tq, int Tk, char* images, int per_head, char* A, typename Window<DH, NT>::Loaded grows,
                                           char* tiles) {
  using W = Window<DH, NT>;
  using R = typename W::R;
  constexpr int CT = W::CT, TILE = W::TILE;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15, nq = (Tq + 15) >> 4;
  char *B = A + W::IMAGE, *C = B + W::IMAGE;
  typename R::Piece kf[NK], vf[NK];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    kf[kt] = R::piece(A + kt * TILE, g, i);
    vf[kt] = R::piece(B + kt * TILE, g, i);
  }
  lds_barrier();
  W::lay(images + W::IMAGE, per_head, grows, Tq);
  lds_barrier();
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 absent;
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = (NK - 1) * 16 + 4 * g + r < Tk ? 0.f : -INFINITY;
  const float c = a.scale * LOG2E;
  f32x4 dk[NK][CT], dv[NK][CT];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) dk[kt][ct] = dv[kt][ct] = zero;
  for (int qt = 0; qt < nq; ++qt) {
    const typename R::Piece qf = R::piece(C + qt * TILE, g, i), gf = R::piece(B + qt * TILE, g, i);
    s16x4 qc[CT], gc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      qc[ct] = R::columns(C + qt * TILE, g, i, ct);
      gc[ct] = R::columns(B + qt * TILE, g, i, ct);
    }
    f32x4 p[NK], dp[NK];
    float d = 0.f, l = 0.f, mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      p[kt] = R::over_channels(kf[kt], qf, kt == NK - 1 ? absent : zero);           // rows = keys, column = query i
      dp[kt] = R::over_channels(vf[kt], gf, zero);
    }
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = larger(mx, p[kt][r]);
    mx = column_max(mx) * c;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[kt][r], c, -mx));
        l += p[kt][r];
        d = __builtin_fmaf(p[kt][r], dp[kt][r], d);
      }
    const bool present = qt * 16 + i < Tq;                                         // no query: P = dS = 0, whatever the keys hold
    const float il = __builtin_amdgcn_rcpf(column_sum(l));
    d = column_sum(d) * il * -a.scale;
    Split ds[NK];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      f32x4 t;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[kt][r] = present ? p[kt][r] * il : 0.f;
        t[r] = present ? p[kt][r] * __builtin_fmaf(dp[kt][r], a.scale, d) : 0.f;
      }
      ds[kt] = gradients(t);
      put_tile(tiles, g, i, probabilities(p[kt]));
      put_tile(tiles + WEIGHT_BYTES, g, i, ds[kt]);
      order_lds();
      const Split pt = turned_tile(tiles, g, i), dt = turned_tile(tiles + WEIGHT_BYTES, g, i);      // queries 4g .. of key i
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        dv[kt][ct] = over_tokens(gc[ct], pt, dv[kt][ct]);
        dk[kt][ct] = over_tokens(qc[ct], dt, dk[kt][ct]);
      }
      order_lds();
    }
    f32x4 dq[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      s16x4 kc[NK];
#pragma unroll
      for (int kt = 0; kt < NK; ++kt) kc[kt] = R::columns(A + kt * TILE, g, i, ct);
      dq[ct] = over_tiles<NK>(kc, ds);
    }
    R::put(C + qt * TILE, g, i, dq);
  }
  order_lds();
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    R::put(A + kt * TILE, g, i, dk[kt]);
    R::put(B + kt * TILE, g, i, dv[kt]);
  }
}

// Windows of up to 16 NT tokens; without a work list (NT = 4) every window, empty ones included.  From two waves per SIMD on, 256 registers at
// most, the matrix instructions write plain vector registers (the backward of 64 channels by 64 tokens needs more: kernel_waves).
template <int DH, int NT, bool BWD> constexpr int window_lds() { return (BWD ? 3 : 2) * Window<DH, NT>::IMAGE + (BWD ? 2 * WEIGHT_BYTES : 0); }
template <int DH, int NT, bool BWD> __device__ __forceinline__ void window_role(const DotArgs& a, int first, int step, int head0, int (*toks)[64], char* images) {
  using W = Window<DH, NT>;
  constexpr int PER_HEAD = window_lds<DH, NT, BWD>();
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* const A = images + w * PER_HEAD;
  for (Walk walk(a, NT == 4 ? 3 : 2, NT == 4 ? 3 : 2, first, step); walk.next(a);) {
    int Tq, Tk;
    walk.tokens(toks, NT * 16, Tq, Tk);
    if (Tq == 0 || Tk == 0) {                            // of all four waves at once: they walk the same windows
      const uint4 z = make_uint4(0u, 0u, 0u, 0u);
      const int col = (head0 + w) * DH * 2;
      if (head0 + w >= a.nhead) continue;
      if (lane < Tq) {
        uint4* o = reinterpret_cast<uint4*>(BWD ? row_of(a.dq, toks[0][lane], a.pdq) + col : row_of(a.o, toks[0][lane], a.po) + col);
        for (int c = 0; c < DH / 8; ++c) o[c] = z;
      }
      if (BWD && lane < Tk) {
        uint4 *p = reinterpret_cast<uint4*>(row_of(a.dk, toks[1][lane], a.pdk) + col),
              *r = reinterpret_cast<uint4*>(row_of(a.dv, toks[1][lane], a.pdv) + col);
        for (int c = 0; c < DH / 8; ++c) { p[c] = z; r[c] = z; }
      }
      continue;
    }
    const typename W::Loaded krows = W::request(a.k, a.pk, toks[1], head0, a.nhead), vrows = W::request(a.v, a.pv, toks[1], head0, a.nhead),
                             qrows = W::request(a.q, a.pq, toks[0], head0, a.nhead);
    constexpr bool LATE = DH * NT >= 128;                // registers: dO is requested when K and V have left theirs
    typename W::Loaded grows;
    if constexpr (BWD && !LATE) grows = W::request(a.g, a.pg, toks[0], head0, a.nhead);
    lds_barrier();                                     // the window before is stored
    W::lay(images, PER_HEAD, krows, Tk);
    W::lay(images + W::IMAGE, PER_HEAD, vrows, Tk);
    if constexpr (BWD) W::lay(images + 2 * W::IMAGE, PER_HEAD, qrows, Tq);
    lds_barrier();
    if constexpr (BWD && LATE) grows = W::request(a.g, a.pg, toks[0], head0, a.nhead);
    const int nk = (Tk + 15) >> 4;
#define ONE(NK)                                                                                                                            \
  if constexpr (BWD) bwd_window<DH, NT, NK>(a, Tq, Tk, images, PER_HEAD, A, grows, A + 3 * W::IMAGE);                              \
  else fwd_window<DH, NT, NK>(a, Tq, Tk, images, PER_HEAD, A, qrows)
    if (nk == 1) { ONE(1); }
    else if (NT == 2 || nk == 2) { ONE(2); }
    else if constexpr (NT == 4) {
      if (nk == 3) { ONE(3); } else { ONE(4); }
    }
#undef ONE
    lds_barrier();
    if constexpr (BWD) {
      W::store(a.dq, a.pdq, toks[0], Tq, head0, a.nhead, images + 2 * W::IMAGE, PER_HEAD);
      W::store(a.dk, a.pdk, toks[1], Tk, head0, a.nhead, images, PER_HEAD);
      W::store(a.dv, a.pdv, toks[1], Tk, head0, a.nhead, images + W::IMAGE, PER_HEAD);
    } else {
      W::store(a.o, a.po, toks[0], Tq, head0, a.nhead, images, PER_HEAD);
    }
  }
}

// ---- windows of at most 16 tokens: a wave per (window, 64 channels), all heads of the 64 channels at once.  Nothing is shared between the
// waves of a workgroup.
constexpr int SMALL_PITCH = 144;           // 128 bytes of a row

// HALF: at most 8 tokens, one load brings a tensor's rows (rows 8 .. 15 then hold them once more)
template <int DH, bool BWD, bool HALF> __device__ __forceinline__ void small_window(const DotArgs& a, const int (*toks)[64], int Tq, int Tk, int head0, char* K) {
  constexpr int HG = 64 / DH, PITCH = SMALL_PITCH, IMAGE = 16 * PITCH, NI = BWD ? 4 : 3;
  using R = Rows<DH, PITCH>;
  constexpr int CT = R::CT;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  char *V = K + IMAGE, *Q = K + 2 * IMAGE, *G = K + 3 * IMAGE;
  const float c = a.scale * LOG2E;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int r8 = lane >> 3, ch = lane & 7;
  const bool in_row = head0 * DH + ch * 8 < a.nhead * DH;
  int col = in_row ? head0 * DH * 2 + ch * 16 : 0;
  asm volatile("" : "+v"(col));             // (seven tensors' addresses of this lane are not worth 14 registers from window to window)
  u32x4 rows[NI][2];
#pragma unroll
  for (int u = 0; u < (HALF ? 1 : 2); ++u) {
    const int tk = toks[1][r8 + 8 * u], tq = toks[0][r8 + 8 * u];
    rows[0][u] = *reinterpret_cast<const u32x4*>(row_of(a.k, tk, a.pk) + col);
    rows[1][u] = *reinterpret_cast<const u32x4*>(row_of(a.v, tk, a.pv) + col);
    rows[2][u] = *reinterpret_cast<const u32x4*>(row_of(a.q, tq, a.pq) + col);
    if constexpr (BWD) rows[3][u] = *reinterpret_cast<const u32x4*>(row_of(a.g, tq, a.pg) + col);
  }
  const u32x4 none = {0u, 0u, 0u, 0u};
  if constexpr (HALF) {
    rows[0][1] = rows[0][0]; rows[2][1] = rows[2][0];
  }
  // slots without a token: zero rows of V and dO, so that a probability of 0 stays one beside an infinity
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    rows[1][u] = (HALF && u) || r8 + 8 * u >= Tk ? none : rows[1][u];
    if constexpr (BWD) rows[3][u] = (HALF && u) || r8 + 8 * u >= Tq ? none : rows[3][u];
  }
#pragma unroll
  for (int t = 0; t < NI; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) *reinterpret_cast<u32x4*>(K + t * IMAGE + (r8 + 8 * u) * PITCH + ch * 16) = rows[t][u];
  order_lds();
  f32x4 absent;
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = 4 * g + r < Tk ? 0.f : -INFINITY;
  if constexpr (!BWD) {
    s16x4 vc[HG][CT];
    Split p[HG];
    f32x4 st[HG];
    float mx[HG], l[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      st[h] = R::over_channels(R::piece(K + h * DH * 2, g, i), R::piece(Q + h * DH * 2, g, i), absent);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) vc[h][ct] = R::columns(V + h * DH * 2, g, i, ct);
    }
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      mx[h] = column_max(larger(larger(st[h][0], st[h][1]), larger(st[h][2], st[h][3]))) * c;
      l[h] = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[h][r], c, -mx[h]));
        l[h] += st[h][r];
      }
      p[h] = probabilities(st[h]);
    }
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      f32x4 o[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] = over_tokens(vc[h][ct], p[h], zero);
      const float il = __builtin_amdgcn_rcpf(column_sum(l[h]));
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] *= il;
      R::put(Q + h * DH * 2, g, i, o);
    }
    order_lds();
    if (in_row) {
#pragma unroll
      for (int u = 0; u < (HALF ? 1 : 2); ++u) {
        const int r = r8 + 8 * u;
        if (r < Tq) *reinterpret_cast<u32x4*>(row_of(a.o, toks[0][r], a.po) + col) = *reinterpret_cast<const u32x4*>(Q + r * PITCH + ch * 16);
      }
    }
  } else {
    s16x4 kc[HG][CT], qc[HG][CT], gc[HG][CT];
    Split ds[HG], pt[HG], dt[HG];            // (the tiles of both kinds share their place in LDS)
    f32x4 p[HG], dp[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      const int at = h * DH * 2;
      p[h] = R::over_channels(R::piece(K + at, g, i), R::piece(Q + at, g, i), absent);
      dp[h] = R::over_channels(R::piece(V + at, g, i), R::piece(G + at, g, i), zero);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        kc[h][ct] = R::columns(K + at, g, i, ct);
        qc[h][ct] = R::columns(Q + at, g, i, ct);
        gc[h][ct] = R::columns(G + at, g, i, ct);
      }
    }
    order_lds();
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      const float mx = column_max(larger(larger(p[h][0], p[h][1]), larger(p[h][2], p[h][3]))) * c;
      float d = 0.f, l = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[h][r], c, -mx));
        l += p[h][r];
        d = __builtin_fmaf(p[h][r], dp[h][r], d);
      }
      const float il = __builtin_amdgcn_rcpf(column_sum(l));
      d = column_sum(d) * il * -a.scale;
      f32x4 t;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[h][r] = i < Tq ? p[h][r] * il : 0.f;                                       // no query: P = dS = 0, whatever the keys hold
        t[r] = i < Tq ? p[h][r] * __builtin_fmaf(dp[h][r], a.scale, d) : 0.f;
      }
      ds[h] = gradients(t);
      put_tile(K + h * WEIGHT_BYTES, g, i, probabilities(p[h]));
    }
    order_lds();
#pragma unroll
    for (int h = 0; h < HG; ++h) pt[h] = turned_tile(K + h * WEIGHT_BYTES, g, i);
    order_lds();
#pragma unroll
    for (int h = 0; h < HG; ++h) put_tile(K + h * WEIGHT_BYTES, g, i, ds[h]);
    order_lds();
#pragma unroll
    for (int h = 0; h < HG; ++h) dt[h] = turned_tile(K + h * WEIGHT_BYTES, g, i);
    order_lds();
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      f32x4 dq[CT], dk[CT], dv[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        dq[ct] = over_tokens(kc[h][ct], ds[h], zero);
        dv[ct] = over_tokens(gc[h][ct], pt[h], zero);
        dk[ct] = over_tokens(qc[h][ct], dt[h], zero);
      }
      R::put(Q + h * DH * 2, g, i, dq);
      R::put(K + h * DH * 2, g, i, dk);
      R::put(V + h * DH * 2, g, i, dv);
    }
    order_lds();
    if (in_row) {
#pragma unroll
      for (int u = 0; u < (HALF ? 1 : 2); ++u) {
        const int r = r8 + 8 * u;
        const char* at = K + r * PITCH + ch * 16;
        if (r < Tq) *reinterpret_cast<u32x4*>(row_of(a.dq, toks[0][r], a.pdq) + col) = *reinterpret_cast<const u32x4*>(at + 2 * IMAGE);
        if (r < Tk) {
          *reinterpret_cast<u32x4*>(row_of(a.dk, toks[1][r], a.pdk) + col) = *reinterpret_cast<const u32x4*>(at);
          *reinterpret_cast<u32x4*>(row_of(a.dv, toks[1][r], a.pdv) + col) = *reinterpret_cast<const u32x4*>(at + IMAGE);
        }
      }
    }
  }
}

template <int DH, bool BWD> constexpr int small_lds() { return (BWD ? 4 : 3) * 16 * SMALL_PITCH; }             // of one wave
template <int DH, bool BWD> __device__ __forceinline__ void small_role(const DotArgs& a, int first, int step, int head0, int (*toks)[64], char* lds) {
  static_assert(64 / DH * WEIGHT_BYTES <= small_lds<DH, BWD>() || !BWD, "the P and dS tiles take the images' place");
  for (Walk walk(a, 1, 0, first, step); walk.next(a);) {
    int Tq, Tk;
    walk.tokens(toks, 16, Tq, Tk);
    if (Tq == 0 || Tk == 0) continue;                    // (the rows are zeroed by those who look for such windows)
    if (Tq <= 8 && Tk <= 8) small_window<DH, BWD, true>(a, toks, Tq, Tk, head0, lds);
    else small_window<DH, BWD, false>(a, toks, Tq, Tk, head0, lds);
    order_lds();
  }
}

// The workgroups of a launch: n4 walk the windows of 33 to 64 tokens (or every window, where there is no list), n2 those of 17 to 32, n1
// the others, each of them with its group of heads; those behind them zero the rows of the windows that are in no list.
struct Roles { int n4, n2, n1, n0, heads, columns; };                   // heads: groups of four; columns: groups of 64 channels
constexpr int ROLE4 = 1, ROLE2 = 2, ROLE1 = 4;
template <int DH, bool BWD, int ROLES> constexpr int kernel_lds() {
  const int l4 = ROLES & ROLE4 ? window_lds<DH, 4, BWD>() : 0, l2 = ROLES & ROLE2 ? window_lds<DH, 2, BWD>() : 0,
            l1 = ROLES & ROLE1 ? small_lds<DH, BWD>() : 0;
  return 4 * (l4 > l2 ? (l4 > l1 ? l4 : l1) : (l2 > l1 ? l2 : l1));
}
template <int DH, bool BWD, int ROLES> constexpr int kernel_waves() {        // waves per SIMD that the registers allow
  if (!BWD) return DH == 16 ? 4 : DH == 32 ? 3 : 2;
  return ROLES & ROLE4 ? (DH == 16 ? 3 : DH == 32 ? 2 : 1) : (DH == 16 ? 4 : DH == 32 ? 3 : 2);
}
template <int DH, bool BWD, int ROLES>
__global__ __launch_bounds__(256, (kernel_waves<DH, BWD, ROLES>())) void dot_kernel(DotArgs a, Roles n, Orphans z) {
  extern __shared__ __attribute__((aligned(16))) char lds_[];
  __shared__ int toks_[4][2][64];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int (*toks)[64] = toks_[w];
  int u = blockIdx.x;
  if constexpr (ROLES & ROLE4) {
    if (u < n.n4 * n.heads) {
      window_role<DH, 4, BWD>(a, u / n.heads, n.n4, u % n.heads * 4, toks, lds_);
      return;
    }
    u -= n.n4 * n.heads;
  }
  if constexpr (ROLES & ROLE2) {
    if (u < n.n2 * n.heads) {
      window_role<DH, 2, BWD>(a, u / n.heads, n.n2, u % n.heads * 4, toks, lds_);
      return;
    }
    u -= n.n2 * n.heads;
  }
  if constexpr (ROLES & ROLE1) {
    if (u < n.n1 * n.columns) {
      small_role<DH, BWD>(a, u / n.columns * 4 + w, n.n1 * 4, u % n.columns * (64 / DH), toks, lds_ + w * small_lds<DH, BWD>());
      return;
    }
    u -= n.n1 * n.columns;
    orphan_role(a, z, u * 4 + w, n.n0 * 4);
  }
}

// Workgroups along the windows: what the windows can need, at most `per_cu` per CU in all -- a little more than what is resident at
// once.  In bfloat16 6 take 111 + 223 us forward and backward at stage 1, 4 take 114 + 228 (the last windows are left to few workgroups),
// 12 take 114 + 230 (some find no window); across frames of stage 2 43 + 86, 41 + 83 and 50 + 96.  Neighbouring windows on the same die
// would share the grids' lines in its L2, but the dense windows are neighbours too: one die would have them all (49 us, not 39, for the
// small and middle windows of stage 2's backward).
unsigned walkers(int64_t windows, int per_group, unsigned gx, int per_cu = 6) {
  const int64_t need = (windows + per_group - 1) / per_group;
  int64_t most = (int64_t)tmae_num_cus() * per_cu / gx;
  if (most < 1) most = 1;
  return (unsigned)(need < most ? need : most);
}
// windows that a class of a work list can hold, where the grids hold rows only: class c > 0 windows have more than 8 * 2^(c-1) tokens of one
// of the two frames.  The list counts entries that are no row as well, so that a class may hold windows that these numbers rule out: one
// workgroup at least walks every class, and a walk goes through the whole of it.
int64_t class_windows(const DotArgs& a, int cls) {
  const int64_t most = (a.mq + a.mk) / (cls == 0 ? 2 : cls == 1 ? 9 : cls == 2 ? 17 : 33);
  return most < 1 ? 1 : most < a.nwin ? most : a.nwin;
}

bool rows_ok(const void* p, int64_t ld, int width, int es) {
  return p && ((uintptr_t)p & 15) == 0 && ld >= width && ld < (1 << 28) && (ld * es) % 16 == 0;
}

int fill(DotArgs& a, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny,
         int nx, int do_shift, float scale, const int32_t* worklist) {
  if (dtype != TMAE_F32 && dtype != TMAE_BF16) return TMAE_EDTYPE;
  if (mq < 0 || mk < 0 || mq > 0x7fffffff || mk > 0x7fffffff || nhead < 1 || nhead > 4096 || (dh != 16 && dh != 32 && dh != 64)) return TMAE_EARG;
  if (!grid_q || !grid_k || batch < 1 || ny < 1 || nx < 1 || (int64_t)ny * nx >= ((int64_t)1 << 31) ||
      (int64_t)batch * ny * nx >= ((int64_t)1 << 31) || !(scale > 0.f) || scale > 2e38f)
    return TMAE_EARG;
  a.Wy = (ny + WIN - 1) / WIN + 1; a.Wx = (nx + WIN - 1) / WIN + 1;
  if (worklist && (a.Wy > 255 || a.Wx > 255 || batch > 32767)) return TMAE_EARG;
  a.nwin = (int64_t)batch * a.Wy * a.Wx;
  if (a.nwin > 0x7fffffff) return TMAE_EARG;
  a.grid_q = grid_q; a.grid_k = grid_k; a.wl = worklist; a.mq = mq; a.mk = mk; a.nhead = nhead; a.batch = batch; a.ny = ny; a.nx = nx;
  a.s = do_shift ? WIN / 2 : WIN;
  a.scale = scale;
  return TMAE_OK;
}

template <class F> void by_head(int dh, F&& f) {
  if (dh == 16) f(std::integral_constant<int, 16>());
  else if (dh == 32) f(std::integral_constant<int, 32>());
  else f(std::integral_constant<int, 64>());
}
template <int DH, bool BWD, int ROLES> int launch_roles(const DotArgs& a, const Orphans& z, int64_t w4, int64_t w2, int64_t w1, hipStream_t stream) {
  constexpr int LDS = kernel_lds<DH, BWD, ROLES>();
  static TmaeLdsAttr attr;
  if (LDS + 2048 > 65536)
    if (int e = tmae_allow_lds(attr, (const void*)dot_kernel<DH, BWD, ROLES>, LDS)) return e;
  Roles n;
  n.heads = (a.nhead + 3) / 4;
  n.columns = (a.nhead * DH + 63) / 64;
  n.n4 = ROLES & ROLE4 ? (int)walkers(w4, 1, n.heads) : 0;
  n.n2 = ROLES & ROLE2 ? (int)walkers(w2, 1, n.heads) : 0;
  n.n1 = ROLES & ROLE1 ? (int)walkers(w1, 4, n.columns) : 0;
  n.n0 = ROLES & ROLE1 && z.row16 ? (int)walkers(a.nwin, 16, 1, 1) : 0;
  const int64_t blocks = (int64_t)(n.n4 + n.n2) * n.heads + (int64_t)n.n1 * n.columns + n.n0;
  if (blocks > 0) hipLaunchKernelGGL((dot_kernel<DH, BWD, ROLES>), dim3((unsigned)blocks), dim3(256), LDS, stream, a, n, z);
  return TMAE_OK;
}
// One launch for all sizes of windows: its workgroups have the registers and the LDS of the largest ones, a second launch costs its own
// tail.  Backward of heads of 16: 217 us in one launch and 219 in two for eight frames at stage 1 (375 k tokens), 11 and 17 for one of 8 k
// tokens; heads of 32 across frames (33 k queries, 131 k keys): 85 and 85.  Of heads of 64 the largest windows leave room for one workgroup
// a CU: 20 and 24 us with 16 k queries and keys, 27 and 27 with 32 k, 49 and 44 with 64 k, 120 and 97 with 188 k.
template <int DH, bool BWD> int launch_bf16(const DotArgs& a, const Orphans& z, hipStream_t stream) {
  const int64_t w4 = a.wl ? class_windows(a, 3) : a.nwin, w2 = class_windows(a, 2), w1 = class_windows(a, 0);
  if (!a.wl) return launch_roles<DH, BWD, ROLE4>(a, z, w4, w2, w1, stream);
  if constexpr (BWD && DH == 64) {
    if (a.mq + a.mk > 32768) {
      const int rc = launch_roles<DH, BWD, ROLE4>(a, z, w4, w2, w1, stream);
      return rc != TMAE_OK ? rc : launch_roles<DH, BWD, ROLE2 | ROLE1>(a, z, w4, w2, w1, stream);
    }
  }
  return launch_roles<DH, BWD, ROLE4 | ROLE2 | ROLE1>(a, z, w4, w2, w1, stream);
}
template <int DH, bool BWD> int launch_f32(const DotArgs& a, const Orphans& z, hipStream_t stream) {
  if (z.row16) hipLaunchKernelGGL(dot_orphan_kernel, dim3(walkers(a.nwin, 4, 1)), dim3(256), 0, stream, a, z);
  constexpr int LDS = ((BWD ? 4 : 3) * Rows32<DH>::IMAGE + 192) * 4;
  static TmaeLdsAttr attr;
  if (LDS + 2048 > 65536)
    if (int e = tmae_allow_lds(attr, (const void*)dot_f32_kernel<DH, BWD>, LDS)) return e;
  Roles32 n;
  n.h4 = a.nhead; n.h2 = (a.nhead + 1) / 2; n.h1 = (a.nhead + 3) / 4;
  // three workgroups a CU for each size: 21 us forward and 48 us backward for a frame of 16 k tokens, 27 and 59 with twelve
  n.n4 = (int)walkers(a.wl ? class_windows(a, 3) : a.nwin, 1, n.h4, 3);
  n.n2 = a.wl ? (int)walkers(class_windows(a, 2), 1, n.h2, 3) : 0;
  n.n1 = a.wl ? (int)walkers(class_windows(a, 0), 1, n.h1, 3) : 0;
  const int64_t blocks = (int64_t)n.n4 * n.h4 + (int64_t)n.n2 * n.h2 + (int64_t)n.n1 * n.h1;
  if (blocks > 0) hipLaunchKernelGGL((dot_f32_kernel<DH, BWD>), dim3((unsigned)blocks), dim3(256), LDS, stream, a, n);
  return TMAE_OK;
}

}  // namespace

int tmae_win_attn_dot_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, int dtype, int64_t mq,
                          int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny, int nx,
                          int do_shift, float scale, void* out, int64_t ldo, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (!rows_ok(q, ldq, d, es) || !rows_ok(out, ldo, d, es) || (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es)))) return TMAE_EARG;
  a.q = q; a.k = k; a.v = v; a.o = out;
  a.pq = (unsigned)(ldq * es); a.pk = (unsigned)(ldk * es); a.pv = (unsigned)(ldv * es); a.po = (unsigned)(ldo * es);
  Orphans z = {};
  if (worklist && (grid_q != grid_k || mq != mk)) z = Orphans{(char*)out, ldo * es, nullptr, nullptr, 0, 0, d * es / 16};
  int failed = TMAE_OK;
  by_head(dh, [&](auto w) {
    constexpr int DH = decltype(w)::value;
    if (dtype == TMAE_BF16) failed = launch_bf16<DH, false>(a, z, (hipStream_t)stream);
    else failed = launch_f32<DH, false>(a, z, (hipStream_t)stream);
  });
  return failed != TMAE_OK ? failed : tmae_launch_status();
}

int tmae_win_attn_dot_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* dout,
                          int64_t lddo, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q,
                          const int32_t* grid_k, int batch, int ny, int nx, int do_shift, float scale, void* dq, int64_t lddq, void* dk,
                          int64_t lddk, void* dv, int64_t lddv, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0 && mk == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (mq && (!rows_ok(q, ldq, d, es) || !rows_ok(dout, lddo, d, es) || !rows_ok(dq, lddq, d, es))) return TMAE_EARG;
  if (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es) || !rows_ok(dk, lddk, d, es) || !rows_ok(dv, lddv, d, es))) return TMAE_EARG;
  a.q = q; a.k = k; a.v = v; a.g = dout; a.dq = dq; a.dk = dk; a.dv = dv;
  a.pq = (unsigned)(ldq * es); a.pk = (unsigned)(ldk * es); a.pv = (unsigned)(ldv * es); a.pg = (unsigned)(lddo * es);
  a.pdq = (unsigned)(lddq * es); a.pdk = (unsigned)(lddk * es); a.pdv = (unsigned)(lddv * es);
  Orphans z = {};
  if (worklist && (grid_q != grid_k || mq != mk)) z = Orphans{(char*)dq, lddq * es, (char*)dk, (char*)dv, lddk * es, lddv * es, d * es / 16};
  int failed = TMAE_OK;
  by_head(dh, [&](auto w) {
    constexpr int DH = decltype(w)::value;
    if (dtype == TMAE_BF16) failed = launch_bf16<DH, true>(a, z, (hipStream_t)stream);
    else failed = launch_f32<DH, true>(a, z, (hipStream_t)stream);
  });
  return failed != TMAE_OK ? failed : tmae_launch_status();
}
