// Scaled-dot-product attention inside 8x8 windows of the token grid.
//
//   P_ij = softmax_j(scale q_i . k_j) over the keys j of the query's window,  o_i = sum_j P_ij v_j;  a window without keys: o_i = 0
//   backward, P recomputed from the saved log2 of the softmax's denominator:
//   dV_j = sum_i P_ij dO_i,  dP_ij = dO_i . v_j,  dS_ij = scale P_ij (dP_ij - sum_j P_ij dP_ij),  dQ_i = sum_j dS_ij k_j,  dK_j = sum_i dS_ij q_i
//
// One wavefront per (window, head), tiles of 16 tokens on the float32 matrix instruction 16x16x4.  Its accumulator layout -- lane
// (g, i) = (lane >> 4, lane & 15) holds rows 4g .. 4g+3 of column i -- is also what its B operand takes, row 4g + r in step r: the
// probabilities go from one product into the next without leaving the registers.  Which of the two products' orders is wanted (the
// query or the key in the column) is had by exchanging the operands.
//
// A slot without a token stands for the window's first one: it is read, its probability is set to 0, and nothing is stored for it.
#include "common.h"
#include <type_traits>

namespace {

constexpr int WIN = 8;
constexpr int WL_HDR = 8;                  // the work list: tmae_window_worklist
constexpr float LOG2E = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct DotArgs {
  const void *q, *k, *v, *g;               // g: dO
  int64_t ldq, ldk, ldv, ldg;
  void *o, *dq, *dk, *dv;
  int64_t ldo, lddq, lddk, lddv;
  float* lse;                              // [mq, nhead]: log2 of sum_j 2^(c q.k_j), c = scale * log2(e)
  const int32_t *grid_q, *grid_k, *wl;
  int64_t mq, mk, nwin;
  int nhead, batch, ny, nx, Wy, Wx, s;
  float scale;
};

struct Window { int Tq, Tk; };

// The window's tokens in cell order, into toks[0] (queries) and toks[1] (keys); slots behind the last token repeat the first one.
// A row number outside the tensors counts as an empty cell.  False: the block has no window.
__device__ __forceinline__ bool find_window(const DotArgs& a, int cls, int (*toks)[64], Window& w) {
  const int lane = threadIdx.x & 63;
  int b, wcy, wcx;
  if (a.wl) {
    const int64_t cnt = a.wl[cls];
    if ((int64_t)blockIdx.x >= cnt || (int64_t)blockIdx.x >= a.nwin) return false;
    const int p = a.wl[WL_HDR + cls * a.nwin + blockIdx.x];
    b = p >> 16; wcx = (p >> 8) & 255; wcy = p & 255;
  } else {
    const unsigned u = blockIdx.x;
    wcy = (int)(u % (unsigned)a.Wy); wcx = (int)((u / (unsigned)a.Wy) % (unsigned)a.Wx); b = (int)(u / (unsigned)(a.Wy * a.Wx));
  }
  const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
  const bool in = b >= 0 && b < a.batch && y >= 0 && y < a.ny && x >= 0 && x < a.nx;
  const int64_t cell = ((int64_t)b * a.ny + y) * a.nx + x;
  int tq = in ? a.grid_q[cell] : -1, tk = in ? a.grid_k[cell] : -1;
  if (tq >= a.mq) tq = -1;
  if (tk >= a.mk) tk = -1;
  const unsigned long long mq = __ballot(tq >= 0), mk = __ballot(tk >= 0), below = (1ull << lane) - 1ull;
  w.Tq = __popcll(mq);
  w.Tk = __popcll(mk);
  const int fq = mq ? __shfl(tq, __ffsll(mq) - 1, 64) : -1, fk = mk ? __shfl(tk, __ffsll(mk) - 1, 64) : -1;
  if (threadIdx.x < 64) {
    if (lane >= w.Tq) toks[0][lane] = fq;
    if (lane >= w.Tk) toks[1][lane] = fk;
    if (tq >= 0) toks[0][__popcll(mq & below)] = tq;
    if (tk >= 0) toks[1][__popcll(mk & below)] = tk;
  }
  return true;
}

// channels KD g .. KD g + KD - 1 of a token's head: what the lane contributes to a product over the channels
template <class T, int KD> __device__ __forceinline__ void load_frag(const T* p, float* f);
template <> __device__ __forceinline__ void load_frag<float, 4>(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
}
template <> __device__ __forceinline__ void load_frag<float, 8>(const float* p, float* f) { load8<float>(p, f); }
template <> __device__ __forceinline__ void load_frag<float, 16>(const float* p, float* f) { load8<float>(p, f); load8<float>(p + 8, f + 8); }
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 4>(const __hip_bfloat16* p, float* f) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xFFFF0000u);
  f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 8>(const __hip_bfloat16* p, float* f) { load8<__hip_bfloat16>(p, f); }
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 16>(const __hip_bfloat16* p, float* f) {
  load8<__hip_bfloat16>(p, f);
  load8<__hip_bfloat16>(p + 8, f + 8);
}
template <class T> __device__ __forceinline__ void store_four(T* p, const f32x4& v) {
#pragma unroll
  for (int r = 0; r < 4; ++r) st_f<T>(p + r, v[r]);
}

__device__ __forceinline__ float lanes4_sum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float lanes4_max(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }

template <int KD> __device__ __forceinline__ f32x4 product(const float* a, const float* b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < KD; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  return c;
}
// c[ct] += (tokens' channels as rows) x (b as columns): rows 16 ct .. +15 of the head's channels, contraction over the tile's tokens
template <class T, int CT>
__device__ __forceinline__ void accumulate(const T* base, int64_t ld, const int* toks, const f32x4& b, f32x4* c, int g, int i) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const T* row = base + (int64_t)toks[4 * g + r] * ld + i;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) c[ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(ld_f<T>(row + 16 * ct), b[r], c[ct], 0, 0, 0);
  }
}
__device__ __forceinline__ void order_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class T, int DH>
__global__ __launch_bounds__(256) void dot_fwd_kernel(DotArgs a, int cls) {
  constexpr int KD = DH / 4, CT = DH / 16;
  __shared__ int toks[2][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  Window win;
  if (!find_window(a, cls, toks, win)) return;
  __syncthreads();
  const int head = blockIdx.y * 4 + w;
  if (head >= a.nhead || win.Tq == 0) return;
  const int hoff = head * DH;
  T* out = (T*)a.o + hoff;
  if (win.Tk == 0) {
    if (lane < win.Tq) {
      T* o = out + (int64_t)toks[0][lane] * a.ldo;
      for (int c = 0; c < DH; ++c) st_f<T>(o + c, 0.f);
      a.lse[(int64_t)toks[0][lane] * a.nhead + head] = 0.f;
    }
    return;
  }
  const T *q = (const T*)a.q + hoff, *k = (const T*)a.k + hoff, *v = (const T*)a.v + hoff;
  const int nq = (win.Tq + 15) >> 4, nk = (win.Tk + 15) >> 4;
  const float c = a.scale * LOG2E;
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tq = toks[0][qt * 16 + i];
    float qf[KD];
    load_frag<T, KD>(q + tq * a.ldq + KD * g, qf);
    f32x4 st[4];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        float kf[KD];
        load_frag<T, KD>(k + (int64_t)toks[1][kt * 16 + i] * a.ldk + KD * g, kf);
        st[kt] = product<KD>(kf, qf);                                  // rows = keys, column = query i
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (kt * 16 + 4 * g + r >= win.Tk) st[kt][r] = -INFINITY;
          mx = fmaxf(mx, st[kt][r]);
        }
      }
    }
    mx = lanes4_max(mx) * c;
    float l = 0.f;
    f32x4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = kt * 16 + 4 * g + r < win.Tk ? __builtin_amdgcn_exp2f(fmaf(st[kt][r], c, -mx)) : 0.f;
          l += p[r];
        }
        accumulate<T, CT>(v, a.ldv, toks[1] + kt * 16, p, o, g, i);      // rows = channels, column = query i
      }
    }
    l = lanes4_sum(l);
    if (qt * 16 + i < win.Tq) {
      const float inv = 1.f / l;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) store_four<T>(out + tq * a.ldo + 16 * ct + 4 * g, o[ct] * inv);
      if (g == 0) a.lse[tq * a.nhead + head] = mx + __builtin_amdgcn_logf(l);          // v_log_f32: the logarithm to base 2
    }
  }
}

template <class T, int DH>
__global__ __launch_bounds__(256) void dot_bwd_kernel(DotArgs a, int cls) {
  constexpr int KD = DH / 4, CT = DH / 16;
  __shared__ int toks[2][64];
  __shared__ float lse[4][64], dot[4][64];               // of the query slots: saved log2 denominator, sum_j P dP
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  Window win;
  if (!find_window(a, cls, toks, win)) return;
  __syncthreads();
  const int head = blockIdx.y * 4 + w;
  if (head >= a.nhead) return;
  const int hoff = head * DH;
  T *dq = (T*)a.dq + hoff, *dk = (T*)a.dk + hoff, *dv = (T*)a.dv + hoff;
  if (win.Tq == 0 || win.Tk == 0) {
    if (lane < win.Tq) {
      T* p = dq + (int64_t)toks[0][lane] * a.lddq;
      for (int c = 0; c < DH; ++c) st_f<T>(p + c, 0.f);
    }
    if (lane < win.Tk) {
      T *p = dk + (int64_t)toks[1][lane] * a.lddk, *r = dv + (int64_t)toks[1][lane] * a.lddv;
      for (int c = 0; c < DH; ++c) { st_f<T>(p + c, 0.f); st_f<T>(r + c, 0.f); }
    }
    return;
  }
  const T *q = (const T*)a.q + hoff, *k = (const T*)a.k + hoff, *v = (const T*)a.v + hoff, *gr = (const T*)a.g + hoff;
  const int nq = (win.Tq + 15) >> 4, nk = (win.Tk + 15) >> 4;
  const float c = a.scale * LOG2E;
  lse[w][lane] = a.lse[(int64_t)toks[0][lane] * a.nhead + head];
  order_lds();
  // dQ: the query in the column
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tq = toks[0][qt * 16 + i];
    const float ls = lse[w][qt * 16 + i];
    float qf[KD], gf[KD];
    load_frag<T, KD>(q + tq * a.ldq + KD * g, qf);
    load_frag<T, KD>(gr + tq * a.ldg + KD * g, gf);
    f32x4 p[4], dp[4], acc[CT];
    float d = 0.f;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        const int64_t tk = toks[1][kt * 16 + i];
        float f[KD];
        load_frag<T, KD>(k + tk * a.ldk + KD * g, f);
        const f32x4 s = product<KD>(f, qf);
        load_frag<T, KD>(v + tk * a.ldv + KD * g, f);
        dp[kt] = product<KD>(f, gf);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[kt][r] = kt * 16 + 4 * g + r < win.Tk ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -ls)) : 0.f;
          d += p[kt][r] * dp[kt][r];
        }
      }
    }
    d = lanes4_sum(d);
    if (g == 0) dot[w][qt * 16 + i] = d;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        f32x4 ds;
#pragma unroll
        for (int r = 0; r < 4; ++r) ds[r] = a.scale * p[kt][r] * (dp[kt][r] - d);
        accumulate<T, CT>(k, a.ldk, toks[1] + kt * 16, ds, acc, g, i);
      }
    }
    if (qt * 16 + i < win.Tq) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) store_four<T>(dq + tq * a.lddq + 16 * ct + 4 * g, acc[ct]);
    }
  }
  order_lds();
  // dK, dV: the key in the column
  for (int kt = 0; kt < nk; ++kt) {
    const int64_t tk = toks[1][kt * 16 + i];
    float kf[KD], vf[KD];
    load_frag<T, KD>(k + tk * a.ldk + KD * g, kf);
    load_frag<T, KD>(v + tk * a.ldv + KD * g, vf);
    f32x4 ak[CT], av[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) ak[ct] = av[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int qt = 0; qt < nq; ++qt) {
      const int64_t tq = toks[0][qt * 16 + i];
      float f[KD];
      load_frag<T, KD>(q + tq * a.ldq + KD * g, f);
      const f32x4 s = product<KD>(f, kf);                               // rows = queries, column = key i
      load_frag<T, KD>(gr + tq * a.ldg + KD * g, f);
      const f32x4 dp = product<KD>(f, vf);
      f32x4 p, ds;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int slot = qt * 16 + 4 * g + r;
        p[r] = slot < win.Tq ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse[w][slot])) : 0.f;
        ds[r] = a.scale * p[r] * (dp[r] - dot[w][slot]);
      }
      accumulate<T, CT>(gr, a.ldg, toks[0] + qt * 16, p, av, g, i);
      accumulate<T, CT>(q, a.ldq, toks[0] + qt * 16, ds, ak, g, i);
    }
    if (kt * 16 + i < win.Tk) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        store_four<T>(dk + tk * a.lddk + 16 * ct + 4 * g, ak[ct]);
        store_four<T>(dv + tk * a.lddv + 16 * ct + 4 * g, av[ct]);
      }
    }
  }
}

// The windows that are in no list: zero rows for queries without a key (out, or dq) and for keys without a query (dk, dv).  One wave per
// window, a lane per cell.
__global__ __launch_bounds__(256) void dot_orphan_kernel(DotArgs a, char* q0, int64_t ldq0, char* k0, int64_t ldk0, char* k1, int64_t ldk1,
                                                        int row16) {
  const int lane = threadIdx.x & 63;
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= a.nwin) return;
  const int wcy = (int)(u % a.Wy), wcx = (int)((u / a.Wy) % a.Wx), b = (int)(u / ((int64_t)a.Wy * a.Wx));
  const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
  const bool in = y >= 0 && y < a.ny && x >= 0 && x < a.nx;
  const int64_t cell = ((int64_t)b * a.ny + y) * a.nx + x;
  int tq = in ? a.grid_q[cell] : -1, tk = in ? a.grid_k[cell] : -1;
  if (tq >= a.mq) tq = -1;
  if (tk >= a.mk) tk = -1;
  const bool some_q = __ballot(tq >= 0) != 0, some_k = __ballot(tk >= 0) != 0;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  if (q0 && !some_k && tq >= 0)
    for (int c = 0; c < row16; ++c) reinterpret_cast<uint4*>(q0 + tq * ldq0)[c] = z;
  if (k0 && !some_q && tk >= 0)
    for (int c = 0; c < row16; ++c) {
      reinterpret_cast<uint4*>(k0 + tk * ldk0)[c] = z;
      reinterpret_cast<uint4*>(k1 + tk * ldk1)[c] = z;
    }
}

// blocks of a work list's class: class c > 0 windows hold more than 8 * 2^(c-1) tokens of one of the two frames
int64_t class_blocks(int cls, int64_t nwin, int64_t mq, int64_t mk) {
  const int64_t most = cls == 0 ? nwin : (mq + mk) / (cls == 1 ? 9 : cls == 2 ? 17 : 33);
  return most < nwin ? most : nwin;
}

bool rows_ok(const void* p, int64_t ld, int width, int es) {
  return p && ((uintptr_t)p & 15) == 0 && ld >= width && (ld * es) % 16 == 0;
}

int fill(DotArgs& a, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny,
         int nx, int do_shift, float scale, const int32_t* worklist) {
  if (dtype != TMAE_F32 && dtype != TMAE_BF16) return TMAE_EDTYPE;
  if (mq < 0 || mk < 0 || mq > 0x7fffffff || mk > 0x7fffffff || nhead < 1 || nhead > 4096 || (dh != 16 && dh != 32 && dh != 64)) return TMAE_EARG;
  if (!grid_q || !grid_k || batch < 1 || ny < 1 || nx < 1 || (int64_t)ny * nx >= ((int64_t)1 << 31) ||
      (int64_t)batch * ny * nx >= ((int64_t)1 << 31) || !(scale > 0.f) || scale > 3e38f)
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

template <class F> void by_head(int dtype, int dh, F&& f) {
  auto with = [&](auto t) {
    using T = decltype(t);
    if (dh == 16) f(T(), std::integral_constant<int, 16>());
    else if (dh == 32) f(T(), std::integral_constant<int, 32>());
    else f(T(), std::integral_constant<int, 64>());
  };
  if (dtype == TMAE_BF16) with(__hip_bfloat16()); else with(0.f);
}
template <class F> void by_class(const DotArgs& a, F&& f) {
  const unsigned gy = (unsigned)((a.nhead + 3) / 4);
  if (!a.wl) { f(dim3((unsigned)a.nwin, gy), 0); return; }
  for (int cls = 3; cls >= 0; --cls) {
    const int64_t blocks = class_blocks(cls, a.nwin, a.mq, a.mk);
    if (blocks > 0) f(dim3((unsigned)blocks, gy), cls);
  }
}

}  // namespace

int tmae_win_attn_dot_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, int dtype, int64_t mq,
                          int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny, int nx,
                          int do_shift, float scale, void* out, int64_t ldo, float* lse, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (!rows_ok(q, ldq, d, es) || !rows_ok(out, ldo, d, es) || !lse || (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es)))) return TMAE_EARG;
  a.q = q; a.ldq = ldq; a.k = k; a.ldk = ldk; a.v = v; a.ldv = ldv; a.o = out; a.ldo = ldo; a.lse = lse;
  if (worklist && grid_q != grid_k)
    hipLaunchKernelGGL(dot_orphan_kernel, dim3(tmae_cdiv(a.nwin, 4)), dim3(256), 0, (hipStream_t)stream, a, (char*)out, ldo * es, nullptr,
                       (int64_t)0, nullptr, (int64_t)0, d * es / 16);
  by_head(dtype, dh, [&](auto t, auto w) {
    by_class(a, [&](dim3 grid, int cls) {
      hipLaunchKernelGGL((dot_fwd_kernel<decltype(t), decltype(w)::value>), grid, dim3(256), 0, (hipStream_t)stream, a, cls);
    });
  });
  return tmae_launch_status();
}

int tmae_win_attn_dot_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* dout,
                          int64_t lddo, const float* lse, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q,
                          const int32_t* grid_k, int batch, int ny, int nx, int do_shift, float scale, void* dq, int64_t lddq, void* dk,
                          int64_t lddk, void* dv, int64_t lddv, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0 && mk == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (mq && (!rows_ok(q, ldq, d, es) || !rows_ok(dout, lddo, d, es) || !rows_ok(dq, lddq, d, es) || !lse)) return TMAE_EARG;
  if (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es) || !rows_ok(dk, lddk, d, es) || !rows_ok(dv, lddv, d, es))) return TMAE_EARG;
  a.q = q; a.ldq = ldq; a.k = k; a.ldk = ldk; a.v = v; a.ldv = ldv; a.g = dout; a.ldg = lddo; a.lse = const_cast<float*>(lse);
  a.dq = dq; a.lddq = lddq; a.dk = dk; a.lddk = lddk; a.dv = dv; a.lddv = lddv;
  if (worklist && grid_q != grid_k)
    hipLaunchKernelGGL(dot_orphan_kernel, dim3(tmae_cdiv(a.nwin, 4)), dim3(256), 0, (hipStream_t)stream, a, (char*)dq, lddq * es,
                       (char*)dk, lddk * es, (char*)dv, lddv * es, d * es / 16);
  by_head(dtype, dh, [&](auto t, auto w) {
    by_class(a, [&](dim3 grid, int cls) {
      hipLaunchKernelGGL((dot_bwd_kernel<decltype(t), decltype(w)::value>), grid, dim3(256), 0, (hipStream_t)stream, a, cls);
    });
  });
  return tmae_launch_status();
}
