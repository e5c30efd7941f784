// Norms before and after a block, with its gate and residual scale.
//
//   z = h w_out / rms(h)   (or h)          rms(v) = sqrt(mean(v^2) + eps)
//   out = x + s g z
//   y = out w_in / rms(out)
//
// and backwards, with r1 = 1 / rms(h), r2 = 1 / rms(out), hat = h r1, unit =
// out r2, b = dy w_in, c2 = mean(b unit):
//   d = dout + r2 (b - unit c2)                       the gradient of out, and dx
//   dz = s g d,  dh = r1 (dz w_out - hat mean(dz w_out hat))   (or dz)
//   dg = s z d,  dw_out = sum_rows dz hat,  dw_in = sum_rows dy unit
//
// d is linear in c2, so the backward pass needs one reduction a row: the sums of
// b unit, s g z d0 and s g z d1 with d0 = dout + r2 b and d1 = r2 unit. r1 and r2
// are kept from the forward pass, `out` is made again in fp32.
//
// Everything is fp32 between a value's load and its one rounding. A row is read once into
// registers (a group of threads a row, NP pieces of 16 bytes each) and every output written
// once. Column sums stay in shared memory over the rows of a group; each group writes its
// part, and a second kernel adds the parts in their order, so that results repeat to the
// bit. Measured on a B200: 16384 x 4096 bf16, both norms and a gate by channel, 114 us
// forward (537 MB, 4.7 TB/s) and 243 us for all of the gradients (805 MB, 3.3 TB/s). Neither
// memory (6.55 TB/s) nor the issue slots (62% and 58% used) are what bounds them: it is
// latency that the warps do not cover. Forwards 29 warps an SM wait for the row's loads
// (a quarter of a warp's cycles), backwards the 16 that registers and column sums allow
// wait for shared memory (a fifth; its pipe is 68% busy) and for each instruction's own
// latency (a fifth).
// Rows of odd length pay for values that lie at no fixed place, and for spills: 4099 x 5001
// f16 72 us for 164 MB, all gradients with norm_out and a gate by channel 306 us, bf16 243.
// Spilled bytes (stores / loads of a thread): shifted rows of two pieces forwards f16 220 /
// 276, bf16 96 / 116 (at the 64 registers of two CTAs an SM), backwards f16 264 / 248, bf16
// 64 / 76, of four pieces backwards f16 634 / 1044, bf16 192 / 436; whole rows of two pieces
// forwards f16 56 / 80, bf16 28 / 36. How much of the time is theirs was not measured.
// Rows longer than 2048 pieces are read again for each step, and their column sums stay in
// global memory: 2048 x 32768 bf16 192 us forward and 1251 us backward.
#include <type_traits>

#include "experts.cuh"

namespace es {
namespace {

constexpr int kNormThreads = 256;  // of a CTA whose rows take fewer
constexpr int kMostThreads = 512;
constexpr unsigned kAll = 0xffffffffu;

struct NormArgs {
  const void* x;
  const void* h;
  const void* w_in;
  const void* w_out;
  const void* gate;
  int64_t x_stride, h_stride, gate_stride, dout_stride, dy_stride;
  int64_t rows, width;
  int gate_kind;
  float scale, eps;
  void* out;
  void* y;
  float* stats;  // (rows, 2): r1, r2
  // backward
  const void* dout;
  const void* dy;
  void* dx;
  void* dh;
  void* dgate;
  float* part;     // (groups, columns, width)
  int in_col, out_col, gate_col;  // which of a group's parts, -1: none
  int columns;
  int tp;          // threads of a row
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Vec {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load(const T* p, int64_t piece) {
  return reinterpret_cast<const Vec<T, VEC>*>(p)[piece];
}

// All values of a piece in fp32 and back: two 16-bit values an instruction.
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Vec<T, VEC>& p, float (&v)[VEC]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {  // a bf16 is the high half of its fp32
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else if constexpr (std::is_same<T, __half>::value && VEC % 2 == 0) {
    const __half2* w = reinterpret_cast<const __half2*>(p.v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 f = __half22float2(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(p.v[i]);
  }
}

// A piece's arithmetic, two values an instruction. Gradients of 16384 x 4096
// bf16: 267 to 243 us, of 65536 x 512: 121 to 110.
#define ES_PAIR(op, ...)                                                                             \
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t" op         \
      "mov.b64 {%0, %1}, c;\n\t}"                                                                   \
      : "=f"(o0), "=f"(o1)                                                                           \
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1) __VA_ARGS__)

__device__ __forceinline__ void mul_pair(float& o0, float& o1, float a0, float a1, float b0, float b1) {
  ES_PAIR("mul.rn.f32x2 c, a, b;\n\t", );
}

__device__ __forceinline__ void fma_pair(float& o0, float& o1, float a0, float a1, float b0, float b1, float c0,
                                         float c1) {
  ES_PAIR("mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 c, a, b, c;\n\t", , "f"(c0), "f"(c1));
}
#undef ES_PAIR

template <int VEC>
__device__ __forceinline__ void mul(float (&a)[VEC], const float (&b)[VEC]) {
  static_assert(VEC % 2 == 0, "pieces hold whole pairs");
#pragma unroll
  for (int i = 0; i < VEC; i += 2) mul_pair(a[i], a[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
}
template <int VEC>
__device__ __forceinline__ void mul(float (&a)[VEC], float s) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) mul_pair(a[i], a[i + 1], a[i], a[i + 1], s, s);
}
// o = a b + c
template <int VEC>
__device__ __forceinline__ void fma(float (&o)[VEC], const float (&a)[VEC], const float (&b)[VEC],
                                    const float (&c)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) fma_pair(o[i], o[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
}
template <int VEC>
__device__ __forceinline__ void fma(float (&o)[VEC], float s, const float (&b)[VEC], const float (&c)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) fma_pair(o[i], o[i + 1], s, s, b[i], b[i + 1], c[i], c[i + 1]);
}
// The even and the odd values' part of a sum of products.
template <int VEC>
__device__ __forceinline__ void dot(float2& sum, const float (&a)[VEC], const float (&b)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) fma_pair(sum.x, sum.y, a[i], a[i + 1], b[i], b[i + 1], sum.x, sum.y);
}

template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, int64_t piece, const float (&v)[VEC]) {
  Vec<T, VEC> o;
  if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC % 2 == 0) {
    __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(o.v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  } else if constexpr (std::is_same<T, __half>::value && VEC % 2 == 0) {
    __half2* w = reinterpret_cast<__half2*>(o.v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(v[i]);
  }
  reinterpret_cast<Vec<T, VEC>*>(p)[piece] = o;
}

// Sums of N values over the tp threads of a group, for all of them. `part` is not
// written again before every thread of the CTA has passed another barrier.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*part)[32], int tp) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(kAll, v[i], o);
  if (tp <= 32) {
    __syncwarp();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tp >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[i][warp] = v[i];
  }
  __syncthreads();
  const int first = warp / nw * nw;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < nw ? part[i][first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(kAll, v[i], o);
  }
}

constexpr float kDown = 2.6469779601696886e-23f;  // 2^-75: squares of the largest values, 2^16 of them and more, are finite

// rsqrtf is off by up to 2 units of fp32 and the width's reciprocal by half of one: fp32
// outputs and gradients are 1.7e-7 off in the norm, torch's elementary operations 1.5e-7.
__device__ __forceinline__ float inv_rms(float sum, float inv_width, float eps) {
  return rsqrtf(fmaf(sum, inv_width, eps));
}

template <typename T, typename W, int VEC, int NP>
__global__ void __launch_bounds__(kMostThreads) norm_kernel(const __grid_constant__ NormArgs p) {
  constexpr bool LONG = NP == 0;  // rows that no group of threads holds are read again for each step
  constexpr int HELD = LONG ? 1 : NP;
  __shared__ float part[4][1][32];
  const int tp = p.tp, c0 = threadIdx.x % tp;
  const int64_t t = blockIdx.x * static_cast<int64_t>(blockDim.x / tp) + threadIdx.x / tp;
  const bool live = t < p.rows;
  const int64_t row = live ? t : 0, pieces = p.width / VEC;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* h = static_cast<const T*>(p.h) + row * p.h_stride;
  const T* gate = static_cast<const T*>(p.gate) + (p.gate_kind == ES_GATE_CHANNEL ? 0 : row * p.gate_stride);
  const W* w_out = static_cast<const W*>(p.w_out);
  const W* w_in = static_cast<const W*>(p.w_in);
  const float width = 1.0f / static_cast<float>(p.width);
  Vec<T, VEC> xv[HELD], hv[HELD];
  float o[HELD][VEC];

  // fn(slot, piece) for this thread's pieces of the row
  auto each = [&](auto fn) {
    if constexpr (LONG) {
      if (live)
        for (int64_t c = c0; c < pieces; c += tp) fn(0, c);
    } else {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (live && c0 + n * tp < pieces) fn(n, static_cast<int64_t>(c0 + n * tp));
    }
  };
  if constexpr (!LONG) {
    each([&](int n, int64_t c) {
      xv[n] = load<T, VEC>(x, c);
      if (p.h) hv[n] = load<T, VEC>(h, c);
    });
  }
  float r1 = 1.0f, r2 = 1.0f;
  auto rms = [&](auto value, float (*buf)[32], float (*again)[32]) {
    float sum[1] = {0.0f};
    each([&](int n, int64_t c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float v = value(n, c, i);
        sum[0] = fmaf(v, v, sum[0]);
      }
    });
    group_sum(sum, buf, tp);
    // squares past the largest value: the same sum of smaller ones. All threads of the
    // CTA decide alike, for the barrier in it.
    if (tp > 32 ? __syncthreads_or(!(sum[0] < INFINITY)) : __any_sync(kAll, !(sum[0] < INFINITY))) {
      float small[1] = {0.0f};
      each([&](int n, int64_t c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float v = value(n, c, i) * kDown;
          small[0] = fmaf(v, v, small[0]);
        }
      });
      group_sum(small, again, tp);
      if (!(sum[0] < INFINITY)) return inv_rms(small[0], width, p.eps * kDown * kDown) * kDown;
    }
    return inv_rms(sum[0], width, p.eps);
  };
  if (p.w_out)
    r1 = rms(
        [&](int n, int64_t c, int i) {
          if constexpr (LONG) return to_f32(load<T, VEC>(h, c).v[i]);
          return to_f32(hv[n].v[i]);
        },
        part[0], part[1]);
  const float token = p.gate_kind == ES_GATE_TOKEN && live ? to_f32(gate[0]) : 1.0f;
  auto residual = [&](int n, int64_t c, float (&v)[VEC]) {  // out, in fp32
    const Vec<T, VEC> xs = LONG ? load<T, VEC>(x, c) : xv[n];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(xs.v[i]);
    if (!p.h) return;
    const Vec<T, VEC> hs = LONG ? load<T, VEC>(h, c) : hv[n];
    float z[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) z[i] = to_f32(hs.v[i]) * r1;
    if (p.w_out) {
      const Vec<W, VEC> w = load<W, VEC>(w_out, c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] *= to_f32(w.v[i]);
    }
    if (p.gate_kind == ES_GATE_CHANNEL || p.gate_kind == ES_GATE_FULL) {
      const Vec<T, VEC> g = load<T, VEC>(gate, c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = fmaf(p.scale * to_f32(g.v[i]), z[i], v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = fmaf(p.scale * token, z[i], v[i]);
    }
  };
  each([&](int n, int64_t c) {
    residual(n, c, o[n]);
    if (p.out) store<T, VEC>(static_cast<T*>(p.out) + t * p.width, c, o[n]);
  });
  if (p.w_in) {
    r2 = rms(
        [&](int n, int64_t c, int i) {
          if constexpr (LONG) {
            if (i == 0) residual(n, c, o[0]);
            return o[0][i];
          }
          return o[n][i];
        },
        part[2], part[3]);
    each([&](int n, int64_t c) {
      if constexpr (LONG) residual(n, c, o[0]);
      const Vec<W, VEC> w = load<W, VEC>(w_in, c);
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = o[n][i] * r2 * to_f32(w.v[i]);
      store<T, VEC>(static_cast<T*>(p.y) + t * p.width, c, v);
    });
  }
  if (p.stats && live && c0 == 0) {
    p.stats[2 * t] = r1;
    p.stats[2 * t + 1] = r2;
  }
}

template <typename T, typename W, int VEC, int NP>
__global__ void __launch_bounds__(kMostThreads) norm_grad_kernel(const __grid_constant__ NormArgs p) {
  constexpr bool LONG = NP == 0;  // column sums of long rows stay in memory, each thread's its own
  constexpr int HELD = LONG ? 1 : NP;
  __shared__ float part[2][3][32];
  const int tp = p.tp, c0 = threadIdx.x % tp, per = blockDim.x / tp;
  const int64_t pieces = p.width / VEC;
  const int64_t group = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / tp;
  const W* w_out = static_cast<const W*>(p.w_out);
  const W* w_in = static_cast<const W*>(p.w_in);
  const float width = static_cast<float>(p.width);
  float* parts = p.part + group * p.columns * p.width;
  float sums[3][HELD][VEC];
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int n = 0; n < HELD; ++n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[k][n][i] = 0.0f;
  if constexpr (LONG)
    for (int k = 0; k < p.columns; ++k)
      for (int64_t c = c0; c < pieces; c += tp)
#pragma unroll
        for (int i = 0; i < VEC; ++i) parts[k * p.width + c * VEC + i] = 0.0f;

  int turn = 0;
  for (int64_t t0 = blockIdx.x * static_cast<int64_t>(per); t0 < p.rows;
       t0 += gridDim.x * static_cast<int64_t>(per), turn ^= 1) {
    const int64_t t = t0 + threadIdx.x / tp;
    const bool live = t < p.rows;
    const int64_t row = live ? t : 0;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* h = static_cast<const T*>(p.h) + row * p.h_stride;
    const T* gate = static_cast<const T*>(p.gate) + (p.gate_kind == ES_GATE_CHANNEL ? 0 : row * p.gate_stride);
    const T* dout = static_cast<const T*>(p.dout) + row * p.dout_stride;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    const float r1 = p.w_out ? p.stats[2 * row] : 1.0f, r2 = p.dy ? p.stats[2 * row + 1] : 0.0f;
    const float token = p.gate_kind == ES_GATE_TOKEN ? to_f32(gate[0]) : 1.0f;
    Vec<T, VEC> xv[HELD], hv[HELD], ov[HELD], yv[HELD], gv[HELD];
    auto fetch = [&](int n, int64_t c) {
      xv[n] = load<T, VEC>(x, c);
      if (p.h) hv[n] = load<T, VEC>(h, c);
      if (p.dout) ov[n] = load<T, VEC>(dout, c);
      if (p.dy) yv[n] = load<T, VEC>(dy, c);
      if (p.gate_kind == ES_GATE_CHANNEL || p.gate_kind == ES_GATE_FULL) gv[n] = load<T, VEC>(gate, c);
    };
    auto each = [&](auto fn) {
      if constexpr (LONG) {
        if (live)
          for (int64_t c = c0; c < pieces; c += tp) {
            fetch(0, c);
            fn(0, c);
          }
      } else {
#pragma unroll
        for (int n = 0; n < NP; ++n)
          if (live && c0 + n * tp < pieces) fn(n, static_cast<int64_t>(c0 + n * tp));
      }
    };
    if constexpr (!LONG) each(fetch);
    struct Terms {
      float hat, z, g, unit, b, d0, d1;
    };
    auto terms = [&](int n, int64_t c, auto use) {  // use(i, the terms of value i)
      Vec<W, VEC> wo, wi;
      if (p.w_out) wo = load<W, VEC>(w_out, c);
      if (p.dy) wi = load<W, VEC>(w_in, c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        Terms e;
        e.g = p.scale * token;
        if (p.gate_kind == ES_GATE_CHANNEL || p.gate_kind == ES_GATE_FULL) e.g = p.scale * to_f32(gv[n].v[i]);
        e.hat = p.h ? to_f32(hv[n].v[i]) * r1 : 0.0f;
        e.z = p.w_out ? e.hat * to_f32(wo.v[i]) : e.hat;
        e.unit = fmaf(e.g, e.z, to_f32(xv[n].v[i])) * r2;
        e.b = p.dy ? to_f32(yv[n].v[i]) * to_f32(wi.v[i]) : 0.0f;
        e.d0 = fmaf(r2, e.b, p.dout ? to_f32(ov[n].v[i]) : 0.0f);
        e.d1 = r2 * e.unit;
        use(i, e);
      }
    };
    float v[3] = {0.0f, 0.0f, 0.0f};
    const bool by_token = p.gate_kind == ES_GATE_TOKEN;
    each([&](int n, int64_t c) {
      terms(n, c, [&](int, const Terms& e) {
        v[0] = fmaf(e.b, e.unit, v[0]);
        const float z = by_token ? e.z : e.g * e.z;
        v[1] = fmaf(z, e.d0, v[1]);
        v[2] = fmaf(z, e.d1, v[2]);
      });
    });
    group_sum(v, part[turn], tp);
    const float c2 = v[0] / width, zd = v[1] - c2 * v[2];
    const float c1 = (by_token ? p.scale * token * zd : zd) / width;
    if (by_token && p.dgate && live && c0 == 0) static_cast<T*>(p.dgate)[t] = from_f32<T>(p.scale * zd);
    each([&](int n, int64_t c) {
      float dx[VEC], dh[VEC], dg[VEC];
      float add[3][VEC];
      terms(n, c, [&](int i, const Terms& e) {
        const float d = e.d0 - c2 * e.d1, dz = e.g * d;
        dx[i] = d;
        dg[i] = p.scale * e.z * d;
        add[0][i] = p.dy ? to_f32(yv[n].v[i]) * e.unit : 0.0f;
        add[1][i] = dz * e.hat;
        dh[i] = dz;
      });
      if (p.w_out) {
        const Vec<W, VEC> wo = load<W, VEC>(w_out, c);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          dh[i] = r1 * (dh[i] * to_f32(wo.v[i]) - to_f32(hv[n].v[i]) * r1 * c1);
      }
      if (p.dx) store<T, VEC>(static_cast<T*>(p.dx) + t * p.width, c, dx);
      if (p.dh) store<T, VEC>(static_cast<T*>(p.dh) + t * p.width, c, dh);
      if (p.dgate && p.gate_kind == ES_GATE_FULL) store<T, VEC>(static_cast<T*>(p.dgate) + t * p.width, c, dg);
#pragma unroll
      for (int i = 0; i < VEC; ++i) add[2][i] = dg[i];
      if constexpr (LONG) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (p.in_col >= 0) parts[p.in_col * p.width + c * VEC + i] += add[0][i];
          if (p.out_col >= 0) parts[p.out_col * p.width + c * VEC + i] += add[1][i];
          if (p.gate_col >= 0) parts[p.gate_col * p.width + c * VEC + i] += add[2][i];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sums[k][n][i] += add[k][i];
      }
    });
  }
  if constexpr (!LONG) {
    const int at[3] = {p.in_col, p.out_col, p.gate_col};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (at[k] < 0) continue;
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (c0 + n * tp < pieces) store<float, VEC>(parts + at[k] * p.width, c0 + n * tp, sums[k][n]);
    }
  }
}

// ------------------------------------------- rows that a group holds, walked
//
// The form for rows of up to 2048 pieces of 16 bytes: a group of threads walks every
// so-many-th row, NP pieces a thread.
//
// SHIFT: rows whose length is no multiple of a piece. Contiguous rows of one length start
// at one phase within their 16 bytes in all tensors, so the pieces are cut at the
// addresses' borders instead, value e of the row being value (e + phase) % VEC of its piece,
// and only a row's first and last piece are read value by value. Weights and column sums
// lie in shared memory with value e at [e % VEC][e / VEC], where no bank is met twice
// whatever the phase.

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// Places of the values of a row's first piece in a column array in shared memory (one piece
// of room on either side); piece c's lie c further on.
template <int VEC, bool SHIFT>
struct Places {
  int at[SHIFT ? VEC : 1];
  __device__ __forceinline__ Places(int phase, int pitch) {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int j = i - phase;
        at[i] = (j & (VEC - 1)) * pitch + (j < 0 ? 0 : 1);
      }
    }
  }
};

template <typename T, bool SHIFT>
__device__ __forceinline__ Vec<T, kVec<T>> load_piece(const T* row, int64_t c, int phase, int64_t width) {
  constexpr int VEC = kVec<T>;
  if constexpr (!SHIFT) {
    return load<T, VEC>(row, c);
  } else {
    const int64_t e = c * VEC - phase;
    if (e >= 0 && e + VEC <= width) return *reinterpret_cast<const Vec<T, VEC>*>(row + e);
    Vec<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.v[i] = e + i >= 0 && e + i < width ? row[e + i] : T(0.0f);
    return v;
  }
}

template <typename T, bool SHIFT>
__device__ __forceinline__ void store_piece(T* row, int64_t c, int phase, int64_t width, const float (&v)[kVec<T>]) {
  constexpr int VEC = kVec<T>;
  if constexpr (!SHIFT) {
    store<T, VEC>(row, c, v);
  } else {
    const int64_t e = c * VEC - phase;
    if (e >= 0 && e + VEC <= width) {
      store<T, VEC>(row + e, 0, v);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (e + i >= 0 && e + i < width) row[e + i] = from_f32<T>(v[i]);
    }
  }
}

// The columns' arrays (norm_out, norm_in, a gate by channel): read where they lie (they
// stay in the L1), or of shifted rows from shared memory. `at` has the first value of the
// piece's place; values are found from it by `get`.
template <typename T, typename W, bool SHIFT>
struct Columns {
  const W* w_out;
  const W* w_in;
  const T* gate;
  int pitch;

  // Copies what there is to `shared` and points there; the CTA's threads together.
  __device__ __forceinline__ void read(const NormArgs& p, uint8_t* shared) {
    w_out = static_cast<const W*>(p.w_out);
    w_in = static_cast<const W*>(p.w_in);
    gate = p.gate_kind == ES_GATE_CHANNEL ? static_cast<const T*>(p.gate) : nullptr;
    pitch = static_cast<int>(p.width / kVec<T>) + 3;
    if constexpr (SHIFT) {
      if (w_out) w_out = copy(w_out, shared, p.width);
      if (w_in) w_in = copy(w_in, shared, p.width);
      if (gate) gate = copy(gate, shared, p.width);
      __syncthreads();
    }
  }
  template <typename V>
  __device__ __forceinline__ const V* copy(const V* from, uint8_t*& shared, int64_t width) {
    constexpr int VEC = kVec<T>;
    V* to = reinterpret_cast<V*>(shared);
    shared += VEC * pitch * sizeof(V);
    for (int i = threadIdx.x; i < VEC * pitch; i += blockDim.x) {
      const int64_t e = static_cast<int64_t>(i % pitch - 1) * VEC + i / pitch;
      to[i] = e >= 0 && e < width ? from[e] : V(0.0f);
    }
    return to;
  }
  template <typename V>
  __device__ __forceinline__ void get(const V* from, int64_t c, const Places<kVec<T>, SHIFT>& places,
                                      float (&v)[kVec<T>]) const {
    constexpr int VEC = kVec<T>;
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = to_f32(from[places.at[i] + static_cast<int>(c)]);
    } else {
      widen(load<V, VEC>(from, c), v);
    }
  }
};

template <typename T, typename W, int NP, bool SHIFT>
__global__ void __launch_bounds__(kMostThreads, NP > 2 ? 1 : 2) norm_rows_kernel(const __grid_constant__ NormArgs p) {
  constexpr int VEC = kVec<T>;
  // a piece's number: 32 bits spare whole rows registers (16384 x 4096 bf16: 120 -> 114 us)
  using Place = typename std::conditional<SHIFT, int64_t, int>::type;
  extern __shared__ __align__(16) uint8_t shared_columns[];
  __shared__ float part[2][4][1][32];
  const int tp = p.tp, c0 = threadIdx.x % tp, per = blockDim.x / tp;
  const float inv_width = 1.0f / static_cast<float>(p.width);
  Columns<T, W, SHIFT> cols;
  cols.read(p, shared_columns);
  const int64_t step = gridDim.x * static_cast<int64_t>(per);
  int64_t t = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / tp;
  int turn = 0;
  for (int64_t t0 = blockIdx.x * static_cast<int64_t>(per); t0 < p.rows; t0 += step, t += step, turn ^= 1) {
    const bool live = t < p.rows;
    const int phase = SHIFT ? static_cast<int>(t * p.width % VEC) : 0;
    const int pieces =
        static_cast<int>(!live ? 0 : SHIFT ? (p.width + phase + VEC - 1) / VEC : p.width / VEC);
    const Places<VEC, SHIFT> places(phase, cols.pitch);
    const T* x = static_cast<const T*>(p.x) + t * p.x_stride;
    const T* h = static_cast<const T*>(p.h) + t * p.h_stride;
    const T* gate = static_cast<const T*>(p.gate) + t * p.gate_stride;
    // fn(slot, piece); the values past a shifted row's ends are zero
    auto each = [&](auto fn) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (c0 + n * tp < pieces) fn(n, Place(c0 + n * tp));
    };
    Vec<T, VEC> xv[NP], hv[NP];
    each([&](int n, Place c) {
      if (p.h) hv[n] = load_piece<T, SHIFT>(h, c, phase, p.width);
      xv[n] = load_piece<T, SHIFT>(x, c, phase, p.width);
    });
    const float token = p.gate_kind == ES_GATE_TOKEN && live ? to_f32(gate[0]) : 1.0f;
    auto rms = [&](auto value, float (*buf)[32], float (*again)[32]) {  // value(slot, fp32 values)
      float2 pair = make_float2(0.0f, 0.0f);
      each([&](int n, Place) {
        float v[VEC];
        value(n, v);
        dot(pair, v, v);
      });
      float sum[1] = {pair.x + pair.y};
      group_sum(sum, buf, tp);
      const bool big = live && !(sum[0] < INFINITY);
      // squares past the largest value: the same sum of smaller ones. All threads of the
      // CTA decide alike, for the barrier in it.
      if (per == 1 ? big : tp > 32 ? __syncthreads_or(big) : __any_sync(kAll, big)) {
        float small[1] = {0.0f};
        each([&](int n, Place) {
          float v[VEC];
          value(n, v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) small[0] = fmaf(v[i] * kDown, v[i] * kDown, small[0]);
        });
        group_sum(small, again, tp);
        if (big) return inv_rms(small[0], inv_width, p.eps * kDown * kDown) * kDown;
      }
      return inv_rms(sum[0], inv_width, p.eps);
    };
    float r1 = 1.0f, r2 = 1.0f, o[NP][VEC];
    if (p.w_out) r1 = rms([&](int n, float (&v)[VEC]) { widen(hv[n], v); }, part[turn][0], part[turn][1]);
    each([&](int n, Place c) {
      widen(xv[n], o[n]);
      if (p.h) {
        float z[VEC], g[VEC];
        widen(hv[n], z);
        mul(z, r1);
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] = token;
        if (p.w_out) {
          float w[VEC];
          cols.get(cols.w_out, c, places, w);
          mul(z, w);
        }
        if (p.gate_kind == ES_GATE_CHANNEL) cols.get(cols.gate, c, places, g);
        if (p.gate_kind == ES_GATE_FULL) widen(load_piece<T, SHIFT>(gate, c, phase, p.width), g);
        // One by one: in pairs the 64 registers spilled, and took 3% longer.
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[n][i] = fmaf(p.scale * g[i], z[i], o[n][i]);
      }
      if (p.out) store_piece<T, SHIFT>(static_cast<T*>(p.out) + t * p.width, c, phase, p.width, o[n]);
    });
    if (p.w_in) {
      r2 = rms(
          [&](int n, float (&v)[VEC]) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = o[n][i];
          },
          part[turn][2], part[turn][3]);
      each([&](int n, Place c) {
        float w[VEC];
        cols.get(cols.w_in, c, places, w);
        mul(o[n], r2);
        mul(w, o[n]);
        store_piece<T, SHIFT>(static_cast<T*>(p.y) + t * p.width, c, phase, p.width, w);
      });
    }
    if (p.stats && live && c0 == 0) {
      p.stats[2 * t] = r1;
      p.stats[2 * t + 1] = r2;
    }
  }
}

// The gradients. Column sums lie in shared memory, a group's own: of shifted rows a value's
// owner changes from row to row, and the row's reduction is a barrier between them.
template <typename T, typename W, int NP, bool SHIFT>
__global__ void __launch_bounds__(kMostThreads) norm_grad_rows_kernel(const __grid_constant__ NormArgs p) {
  constexpr int VEC = kVec<T>;
  extern __shared__ __align__(16) uint8_t shared_columns[];
  __shared__ float part[2][3][32];
  const int tp = p.tp, c0 = threadIdx.x % tp, per = blockDim.x / tp, pitch = static_cast<int>(p.width / VEC) + 3;
  const float inv_width = 1.0f / static_cast<float>(p.width);
  const int column = VEC * pitch;  // floats of a column sum
  float* const all = reinterpret_cast<float*>(shared_columns);
  float* const sums = all + threadIdx.x / tp * p.columns * column;
  Columns<T, W, SHIFT> cols;
  cols.read(p, shared_columns + static_cast<size_t>(per) * p.columns * column * sizeof(float));
  for (int i = threadIdx.x; i < per * p.columns * column; i += blockDim.x) all[i] = 0.0f;
  __syncthreads();
  auto add = [&](int k, int64_t c, const Places<VEC, SHIFT>& places, const float (&v)[VEC]) {
    float* to = sums + k * column;
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) to[places.at[i] + static_cast<int>(c)] += v[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        float4* at = reinterpret_cast<float4*>(to + c * VEC + i);
        float4 s = *at;
        s.x += v[i];
        s.y += v[i + 1];
        s.z += v[i + 2];
        s.w += v[i + 3];
        *at = s;
      }
    }
  };
  const int64_t step = gridDim.x * static_cast<int64_t>(per);
  int64_t t = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / tp;
  int turn = 0;
  const bool by_token = p.gate_kind == ES_GATE_TOKEN;
  for (int64_t t0 = blockIdx.x * static_cast<int64_t>(per); t0 < p.rows; t0 += step, t += step, turn ^= 1) {
    const bool live = t < p.rows;
    const int64_t row = live ? t : 0;
    const int phase = SHIFT ? static_cast<int>(t * p.width % VEC) : 0;
    const int64_t pieces = !live ? 0 : SHIFT ? (p.width + phase + VEC - 1) / VEC : p.width / VEC;
    const Places<VEC, SHIFT> places(phase, pitch);
    const T* gate = static_cast<const T*>(p.gate) + row * p.gate_stride;
    auto each = [&](auto fn) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (c0 + n * tp < pieces) fn(n, static_cast<int64_t>(c0 + n * tp));
    };
    Vec<T, VEC> xv[NP], hv[NP], ov[NP], yv[NP];
    each([&](int n, int64_t c) {
      xv[n] = load_piece<T, SHIFT>(static_cast<const T*>(p.x) + t * p.x_stride, c, phase, p.width);
      if (p.h) hv[n] = load_piece<T, SHIFT>(static_cast<const T*>(p.h) + t * p.h_stride, c, phase, p.width);
      if (p.dout) ov[n] = load_piece<T, SHIFT>(static_cast<const T*>(p.dout) + t * p.dout_stride, c, phase, p.width);
      if (p.dy) yv[n] = load_piece<T, SHIFT>(static_cast<const T*>(p.dy) + t * p.dy_stride, c, phase, p.width);
    });
    if (tp > 64 && (c0 & 7) == 0 && t + step < p.rows) {
      // the next row towards L2, a lane a line of 128 bytes: few rows are in flight (16384 x
      // 4096 fp32: 400 -> 329 us; rows of a warp or two have enough, and lose 4%)
      auto ahead = [&](const void* base, int64_t stride) {
        const T* from = static_cast<const T*>(base) + (t + step) * stride;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int64_t e = static_cast<int64_t>(c0 + n * tp) * VEC;
          if (e < p.width) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + e));
        }
      };
      ahead(p.x, p.x_stride);
      if (p.h) ahead(p.h, p.h_stride);
      if (p.gate_kind == ES_GATE_FULL) ahead(p.gate, p.gate_stride);
      if (p.dout) ahead(p.dout, p.dout_stride);
      if (p.dy) ahead(p.dy, p.dy_stride);
    }
    const float r1 = p.w_out ? p.stats[2 * row] : 1.0f, r2 = p.dy ? p.stats[2 * row + 1] : 0.0f;
    const float token = by_token ? to_f32(gate[0]) : 1.0f;
    // scale times the gate, and z, of a piece
    auto branch = [&](int n, int64_t c, float (&g)[VEC], float (&z)[VEC]) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        g[i] = token;
        z[i] = 0.0f;
      }
      if (p.h) widen(hv[n], z);
      mul(z, r1);
      if (p.gate_kind == ES_GATE_CHANNEL) cols.get(cols.gate, c, places, g);
      if (p.gate_kind == ES_GATE_FULL) widen(load_piece<T, SHIFT>(gate, c, phase, p.width), g);
      mul(g, p.scale);
      if (p.w_out) {
        float w[VEC];
        cols.get(cols.w_out, c, places, w);
        mul(z, w);
      }
    };
    // unit, b and d0 of a piece; of more than two pieces they are made twice instead of held
    constexpr bool HOLD = NP <= 2;
    float unit[HOLD ? NP : 1][VEC], d0[HOLD ? NP : 1][VEC];
    float2 pair[3] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    auto terms = [&](int n, int64_t c, const float (&g)[VEC], const float (&z)[VEC], float (&u)[VEC], float (&d)[VEC],
                     float (&b)[VEC]) {
      widen(xv[n], u);
      fma(u, g, z, u);
      mul(u, r2);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        d[i] = 0.0f;
        b[i] = 0.0f;
      }
      if (p.dout) widen(ov[n], d);
      if (p.dy) {
        float y[VEC];
        widen(yv[n], y);
        cols.get(cols.w_in, c, places, b);
        mul(b, y);
        fma(d, r2, b, d);
      }
    };
    each([&](int n, int64_t c) {
      float g[VEC], z[VEC], b[VEC];
      branch(n, c, g, z);
      float(&u)[VEC] = unit[HOLD ? n : 0];
      float(&d)[VEC] = d0[HOLD ? n : 0];
      terms(n, c, g, z, u, d, b);
      if (!by_token) mul(z, g);
      dot(pair[0], b, u);
      dot(pair[1], z, d);
      dot(pair[2], z, u);
    });
    float v[3] = {pair[0].x + pair[0].y, pair[1].x + pair[1].y, pair[2].x + pair[2].y};
    group_sum(v, part[turn], tp);
    const float c2 = v[0] * inv_width * r2, zd = v[1] - c2 * v[2];
    const float c1 = (by_token ? p.scale * token * zd : zd) * inv_width;
    if (by_token && p.dgate && live && c0 == 0) static_cast<T*>(p.dgate)[t] = from_f32<T>(p.scale * zd);
    each([&](int n, int64_t c) {
      float g[VEC], z[VEC], d[VEC];
      branch(n, c, g, z);
      float(&u)[VEC] = unit[HOLD ? n : 0];
      if constexpr (!HOLD) {
        float b[VEC];
        terms(n, c, g, z, u, d0[0], b);
      }
      fma(d, -c2, u, d0[HOLD ? n : 0]);
      if (p.dx) store_piece<T, SHIFT>(static_cast<T*>(p.dx) + t * p.width, c, phase, p.width, d);
      if (p.in_col >= 0) {
        float a[VEC];
        widen(yv[n], a);
        mul(a, u);
        add(p.in_col, c, places, a);
      }
      mul(z, d);
      mul(z, p.scale);  // the gate's gradient
      mul(d, g);        // z's
      if (p.gate_col >= 0) add(p.gate_col, c, places, z);
      if (p.dgate && p.gate_kind == ES_GATE_FULL)
        store_piece<T, SHIFT>(static_cast<T*>(p.dgate) + t * p.width, c, phase, p.width, z);
      if (p.w_out) {
        float w[VEC], hat[VEC];
        cols.get(cols.w_out, c, places, w);
        widen(hv[n], hat);
        mul(hat, r1);
        if (p.out_col >= 0) {
          float a[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) a[i] = d[i];
          mul(a, hat);
          add(p.out_col, c, places, a);
        }
        mul(d, w);
        fma(d, -c1, hat, d);
        mul(d, r1);
      }
      if (p.dh) store_piece<T, SHIFT>(static_cast<T*>(p.dh) + t * p.width, c, phase, p.width, d);
    });
  }
  __syncthreads();
  float* parts = p.part + (blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / tp) * p.columns * p.width;
  for (int k = 0; k < p.columns; ++k)
    for (int64_t e = c0; e < p.width; e += tp)
      parts[k * p.width + e] = sums[k * column + (SHIFT ? (e % VEC) * pitch + e / VEC + 1 : e)];
}

// Adds the groups' parts of each column in their order: 32 columns by 32 slices of the
// groups a CTA, the slices' sums added in their order (296 groups of 3 x 4096: 16 us with 8).
struct SumArgs {
  const float* part;
  int64_t groups, width;
  int columns;
  void* out[3];
  int dtype[3];
};

constexpr int kSlices = 32;

__global__ void __launch_bounds__(32 * kSlices) column_sum_kernel(const __grid_constant__ SumArgs p) {
  __shared__ float slices[kSlices][32];
  const int64_t n = p.columns * p.width, at = blockIdx.x * 32LL + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  float sum = 0.0f;
  if (at < n) {
    const int64_t from = p.groups * slice / kSlices, to = p.groups * (slice + 1) / kSlices;
#pragma unroll 4
    for (int64_t g = from; g < to; ++g) sum += p.part[g * n + at];
  }
  slices[slice][threadIdx.x & 31] = sum;
  __syncthreads();
  if (slice || at >= n) return;
#pragma unroll
  for (int s = 1; s < kSlices; ++s) sum += slices[s][threadIdx.x];
  const int k = static_cast<int>(at / p.width);
  const int64_t c = at - k * p.width;
  if (p.dtype[k] == ES_BF16)
    static_cast<__nv_bfloat16*>(p.out[k])[c] = __float2bfloat16(sum);
  else if (p.dtype[k] == ES_F16)
    static_cast<__half*>(p.out[k])[c] = __float2half(sum);
  else
    static_cast<float*>(p.out[k])[c] = sum;
}

// Threads of a row (a multiple of 32) and pieces that each holds, a power of two up
// to `most`; 0 pieces: a row that no 512 threads hold.
struct RowForm {
  int tp, np;
  int groups() const { return tp < kNormThreads ? kNormThreads / tp : 1; }  // of a CTA
  int threads() const { return tp * groups(); }
};

RowForm row_form(int64_t pieces, int most) {
  for (int threads = kNormThreads; threads <= kMostThreads; threads *= 2)
    for (int np = 1; np <= most; np *= 2) {
      const int64_t tp = pieces > 0 ? (pieces + 32 * np - 1) / (32 * np) * 32 : 32;
      if (tp <= threads) return RowForm{static_cast<int>(tp), np};
    }
  return RowForm{kMostThreads, 0};
}

// Groups of threads that walk the rows, `resident` threads an SM.
int64_t walking_groups(int64_t rows, const RowForm& f, int resident) {
  const int64_t per = f.groups(), ctas = (rows + per - 1) / per, most = kSMs * (resident / f.threads());
  return (ctas < most ? ctas : most) * per;
}

// The general backward form's.
int64_t grad_groups(int64_t rows, const RowForm& f) { return walking_groups(rows, f, kMostThreads); }

// The walked form's: with few rows a piece a thread while 512 threads hold the row; with
// many two, since what a warp does for a row (its reductions) costs as much as a piece.
RowForm walked_form(int64_t pieces, int64_t rows) {
  for (int np = rows < 4 * kSMs ? 1 : 2; np <= 4; np *= 2) {
    const int64_t tp = pieces > 0 ? (pieces + 32 * np - 1) / (32 * np) * 32 : 32;
    if (tp <= kMostThreads) {
      while (np > 1 && np * 16 >= pieces) np /= 2;  // rows that fewer pieces a lane hold
      return RowForm{static_cast<int>(tp), np};
    }
  }
  return RowForm{kMostThreads, 0};
}

// Shared memory of the columns (dynamic): the most, and what a launch may have without a
// raised limit, which counts a kernel's own 768 or 1024 bytes too.
constexpr size_t kMostColumnsSmem = 200 * 1024, kFreeColumnsSmem = 47 * 1024;

size_t columns_bytes(int64_t width, int vec, size_t bytes) {
  return static_cast<size_t>(vec) * (width / vec + 3) * bytes;
}

// Bytes of one channel of the arrays that shifted rows keep in shared memory.
size_t array_bytes(const NormArgs& p, size_t weight, size_t value) {
  return ((p.w_in != nullptr) + (p.w_out != nullptr)) * weight + (p.gate_kind == ES_GATE_CHANNEL ? value : 0);
}

// Raises a kernel's limit of shared memory, once a device.
template <typename K>
int raise_smem(K kernel, std::atomic<bool> (&raised)[kMaxAttrDevices]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ES_ERR_CUDA;
  const bool tracked = dev >= 0 && dev < kMaxAttrDevices;
  if (tracked && raised[dev].load(std::memory_order_relaxed)) return ES_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostColumnsSmem)) !=
      cudaSuccess)
    return ES_ERR_CUDA;
  if (tracked) raised[dev].store(true, std::memory_order_relaxed);
  return ES_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How the rows lie: in whole pieces of 16 bytes, all at one phase within them, or neither.
enum Lie { kWhole, kPhase, kAny };

Lie lie_of(const NormArgs& p, int esz) {
  const int64_t vec = 16 / esz;
  const bool full = p.gate_kind == ES_GATE_FULL;
  if (!(aligned16(p.x) && aligned16(p.h) && aligned16(p.out) && aligned16(p.y) && aligned16(p.dout) &&
        aligned16(p.dy) && aligned16(p.dx) && aligned16(p.dh) && (!full || (aligned16(p.gate) && aligned16(p.dgate)))))
    return kAny;
  if (p.width % vec == 0 && p.x_stride % vec == 0 && p.h_stride % vec == 0 && (!full || p.gate_stride % vec == 0) &&
      p.dout_stride % vec == 0 && p.dy_stride % vec == 0 && aligned16(p.w_in) && aligned16(p.w_out) &&
      (p.gate_kind != ES_GATE_CHANNEL || aligned16(p.gate)) && aligned16(p.part))
    return kWhole;
  const bool one = p.x_stride == p.width && (!p.h || p.h_stride == p.width) && (!full || p.gate_stride == p.width) &&
                   (!p.dout || p.dout_stride == p.width) && (!p.dy || p.dy_stride == p.width);
  return one ? kPhase : kAny;
}

// fn(integral_constant<pieces>)
template <int MOST, typename Fn>
int by_pieces(int np, Fn fn) {
  if (np == 0) return fn(std::integral_constant<int, 0>{});
  if constexpr (MOST > 1)
    if (np < MOST) return by_pieces<MOST / 2>(np, fn);
  return fn(std::integral_constant<int, MOST>{});
}

template <typename T, typename W, bool SHIFT>
int forward_rows(NormArgs& p, const RowForm& f, size_t smem, cudaStream_t s) {
  p.tp = f.tp;
  const unsigned blocks = static_cast<unsigned>(walking_groups(p.rows, f, 2 * kMostThreads) / f.groups());
  return by_pieces<4>(f.np, [&](auto np) {
    constexpr int NP = decltype(np)::value;
    if constexpr (NP > 0) {
      static std::atomic<bool> raised[kMaxAttrDevices];
      if (smem > kFreeColumnsSmem) ES_TRY(raise_smem(norm_rows_kernel<T, W, NP, SHIFT>, raised));
      ES_LAUNCH((norm_rows_kernel<T, W, NP, SHIFT>), blocks, f.threads(), smem, s, p);
    }
    return static_cast<int>(ES_OK);
  });
}

template <typename T, typename W>
int forward(NormArgs& p, cudaStream_t s) {
  constexpr int VEC = kVec<T>;
  const Lie lie = lie_of(p, sizeof(T));
  const RowForm f = walked_form(lie == kPhase ? (p.width + 2 * VEC - 2) / VEC : p.width / VEC, p.rows);
  const size_t smem = lie == kPhase ? columns_bytes(p.width, VEC, array_bytes(p, sizeof(W), sizeof(T))) : 0;
  // Odd rows of 16 bits, two pieces a thread, that are added and normalised once after it:
  // value by value 4099 x 5001 f16 is 72 us for 81 in shifted pieces, 13324 x 1501 68 for 80,
  // 38387 x 521 87 for 126. With norm_out, or without h, neither is faster throughout (19980
  // x 1001 95 for 83, 3332 x 6001 81 for 94); with a gate by channel (4099 x 5001 104 for 96),
  // one of each value's (152 for 112) or fp32 (94 for 76) shifted pieces are.
  const bool by_value = lie == kPhase && sizeof(T) == 2 && f.np == 2 && p.h && p.w_in && !p.w_out &&
                        (p.gate_kind == ES_GATE_NONE || p.gate_kind == ES_GATE_TOKEN);
  if (f.np && lie != kAny && !by_value && smem <= kMostColumnsSmem)
    return lie == kWhole ? forward_rows<T, W, false>(p, f, smem, s) : forward_rows<T, W, true>(p, f, smem, s);
  const RowForm r = lie == kWhole ? RowForm{kMostThreads, 0} : row_form(p.width, 16);
  p.tp = r.tp;
  const int64_t per = r.groups();
  const unsigned blocks = static_cast<unsigned>((p.rows + per - 1) / per);
  if (lie == kWhole) {
    ES_LAUNCH((norm_kernel<T, W, VEC, 0>), blocks, r.threads(), 0, s, p);
    return ES_OK;
  }
  return by_pieces<16>(r.np, [&](auto np) {
    ES_LAUNCH((norm_kernel<T, W, 1, decltype(np)::value>), blocks, r.threads(), 0, s, p);
    return static_cast<int>(ES_OK);
  });
}

template <typename T, typename W, bool SHIFT>
int backward_rows(NormArgs& p, const RowForm& f, int64_t groups, size_t smem, cudaStream_t s) {
  p.tp = f.tp;
  return by_pieces<4>(f.np, [&](auto np) {
    constexpr int NP = decltype(np)::value;
    if constexpr (NP > 0) {
      static std::atomic<bool> raised[kMaxAttrDevices];
      if (smem > kFreeColumnsSmem) ES_TRY(raise_smem(norm_grad_rows_kernel<T, W, NP, SHIFT>, raised));
      ES_LAUNCH((norm_grad_rows_kernel<T, W, NP, SHIFT>), static_cast<unsigned>(groups / f.groups()), f.threads(),
                smem, s, p);
    }
    return static_cast<int>(ES_OK);
  });
}

template <typename T, typename W>
int backward(NormArgs& p, const SumArgs& sums, cudaStream_t s) {
  constexpr int VEC = kVec<T>;
  const Lie lie = lie_of(p, sizeof(T));
  const RowForm f = walked_form(lie == kPhase ? (p.width + 2 * VEC - 2) / VEC : p.width / VEC, p.rows);
  const size_t smem = columns_bytes(p.width, VEC, p.columns * f.groups() * sizeof(float) +
                                                      (lie == kPhase ? array_bytes(p, sizeof(W), sizeof(T)) : 0));
  int64_t groups;
  if (f.np && lie != kAny && smem <= kMostColumnsSmem) {
    groups = walking_groups(p.rows, f, kMostThreads);
    ES_TRY((lie == kWhole ? backward_rows<T, W, false>(p, f, groups, smem, s)
                          : backward_rows<T, W, true>(p, f, groups, smem, s)));
  } else {
    const RowForm r = lie == kWhole ? RowForm{kMostThreads, 0} : row_form(p.width, 16);
    p.tp = r.tp;
    groups = grad_groups(p.rows, r);
    const unsigned blocks = static_cast<unsigned>(groups / r.groups());
    if (lie == kWhole)
      ES_LAUNCH((norm_grad_kernel<T, W, VEC, 0>), blocks, r.threads(), 0, s, p);
    else
      ES_TRY(by_pieces<16>(r.np, [&](auto np) {
        ES_LAUNCH((norm_grad_kernel<T, W, 1, decltype(np)::value>), blocks, r.threads(), 0, s, p);
        return static_cast<int>(ES_OK);
      }));
  }
  if (!p.columns) return ES_OK;
  SumArgs a = sums;
  a.groups = groups;
  ES_LAUNCH(column_sum_kernel, static_cast<unsigned>((p.columns * p.width + 31) / 32), 32 * kSlices, 0, s, a);
  return ES_OK;
}

int check_norm(const NormArgs& p, int dtype, int weight_dtype) {
  if (p.rows < 0 || p.width < 0 || p.gate_kind < ES_GATE_NONE || p.gate_kind > ES_GATE_FULL) return ES_ERR_INVALID;
  if ((p.gate_kind != ES_GATE_NONE) != (p.gate != nullptr) || (!p.h && (p.gate || p.w_out || !p.w_in)))
    return ES_ERR_INVALID;
  if (p.rows > 0x7fffff00LL || p.width > 0x7fffff00LL / 4) return ES_ERR_UNSUPPORTED;
  if (dtype != ES_F32 && dtype != ES_BF16 && dtype != ES_F16) return ES_ERR_UNSUPPORTED;
  if (weight_dtype != dtype && weight_dtype != ES_F32) return ES_ERR_UNSUPPORTED;
  return ES_OK;
}

// fn<T, W>() by types
#define ES_NORM_CALL(fn, ...)                                                                     \
  ES_BY_TYPE(dtype, return weight_dtype == dtype ? fn<T, T>(__VA_ARGS__) : fn<T, float>(__VA_ARGS__))

}  // namespace
}  // namespace es

using namespace es;

extern "C" int es_residual_norm(const void* x, int64_t x_stride, const void* h, int64_t h_stride, int dtype,
                                int64_t num_rows, int64_t width, const void* norm_in, const void* norm_out,
                                int weight_dtype, const void* gate, int gate_kind, int64_t gate_stride, float scale,
                                float eps, void* out, void* y, float* stats, void* stream) {
  NormArgs p{};
  p.x = x;
  p.h = h;
  p.x_stride = x_stride;
  p.h_stride = h_stride;
  p.w_in = norm_in;
  p.w_out = norm_out;
  p.gate = gate;
  p.gate_kind = gate_kind;
  p.gate_stride = gate_stride;
  p.rows = num_rows;
  p.width = width;
  p.scale = scale;
  p.eps = eps;
  p.out = out;
  p.y = y;
  p.stats = stats;
  if (num_rows < 0 || width < 0) return ES_ERR_INVALID;
  if (num_rows == 0 || width == 0) return ES_OK;
  ES_TRY(check_norm(p, dtype, weight_dtype));
  if (!x || (h && !out) || (norm_in && !y)) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  ES_NORM_CALL(forward, p, s);
  return ES_ERR_UNSUPPORTED;
}

// Column sums that the gradients given need.
static int norm_columns(const void* dnorm_in, const void* dnorm_out, const void* dgate, int gate_kind) {
  return (dnorm_in ? 1 : 0) + (dnorm_out ? 1 : 0) + (dgate && gate_kind == ES_GATE_CHANNEL ? 1 : 0);
}

extern "C" size_t es_residual_norm_grad_workspace_size(int dtype, int64_t num_rows, int64_t width, int num_columns) {
  if (num_rows <= 0 || width <= 0 || num_columns <= 0) return 0;
  // as many groups as the form has that takes most, by addresses that are not known here
  const int vec = dtype == ES_F32 ? 4 : 8;
  int64_t groups = grad_groups(num_rows, row_form(width, 16));
  for (const RowForm f : {RowForm{kMostThreads, 0}, walked_form(width / vec, num_rows),
                          walked_form((width + 2 * vec - 2) / vec, num_rows)}) {
    const int64_t n = walking_groups(num_rows, f, kMostThreads);
    if (n > groups) groups = n;
  }
  return static_cast<size_t>(groups) * num_columns * width * sizeof(float);
}

extern "C" int es_residual_norm_grad(const void* x, int64_t x_stride, const void* h, int64_t h_stride, int dtype,
                                     int64_t num_rows, int64_t width, const void* norm_in, const void* norm_out,
                                     int weight_dtype, const void* gate, int gate_kind, int64_t gate_stride,
                                     float scale, const float* stats, const void* dout, int64_t dout_stride,
                                     const void* dy, int64_t dy_stride, void* dx, void* dh, void* dgate,
                                     void* dnorm_in, void* dnorm_out, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  NormArgs p{};
  p.x = x;
  p.h = h;
  p.x_stride = x_stride;
  p.h_stride = h_stride;
  p.w_in = norm_in;
  p.w_out = norm_out;
  p.gate = gate;
  p.gate_kind = gate_kind;
  p.gate_stride = gate_stride;
  p.rows = num_rows;
  p.width = width;
  p.scale = scale;
  p.stats = const_cast<float*>(stats);
  p.dout = dout;
  p.dout_stride = dout ? dout_stride : 0;
  p.dy = dy;
  p.dy_stride = dy ? dy_stride : 0;
  p.dx = dx;
  p.dh = dh;
  p.dgate = dgate;
  if (num_rows < 0 || width < 0) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (width == 0) {  // a gate by token still has a value a row: a sum over no channels
    if (dgate && gate_kind == ES_GATE_TOKEN && num_rows > 0 &&
        cudaMemsetAsync(dgate, 0, num_rows * (dtype == ES_F32 ? 4 : 2), s) != cudaSuccess)
      return ES_ERR_CUDA;
    return ES_OK;
  }
  if (num_rows > 0) {  // tensors without values have no addresses
    ES_TRY(check_norm(p, dtype, weight_dtype));
    if ((dy && !norm_in) || (dh && !h) || (dgate && !gate) || (dnorm_in && !norm_in) || (dnorm_out && !norm_out) ||
        !x || ((norm_out || dy) && !stats))
      return ES_ERR_INVALID;
  }
  SumArgs sums{};
  sums.width = width;
  p.in_col = p.out_col = p.gate_col = -1;
  auto column = [&](int& col, void* out, int type) {
    col = sums.columns;
    sums.out[sums.columns] = out;
    sums.dtype[sums.columns++] = type;
  };
  if (dnorm_in && dy) column(p.in_col, dnorm_in, weight_dtype);
  if (dnorm_out) column(p.out_col, dnorm_out, weight_dtype);
  if (dgate && gate_kind == ES_GATE_CHANNEL) column(p.gate_col, dgate, dtype);
  p.columns = sums.columns;
  auto clear = [&](void* out, int type) {
    return cudaMemsetAsync(out, 0, width * (type == ES_F32 ? 4 : 2), s) == cudaSuccess ? ES_OK : ES_ERR_CUDA;
  };
  if (num_rows == 0) {  // sums of nothing
    for (int k = 0; k < sums.columns; ++k) ES_TRY(clear(sums.out[k], sums.dtype[k]));
    if (dnorm_in && !dy) ES_TRY(clear(dnorm_in, weight_dtype));
    return ES_OK;
  }
  if (workspace_bytes < es_residual_norm_grad_workspace_size(
                            dtype, num_rows, width, norm_columns(dnorm_in, dnorm_out, dgate, gate_kind)))
    return ES_ERR_WORKSPACE;
  if (p.columns && !workspace) return ES_ERR_WORKSPACE;
  p.part = static_cast<float*>(workspace);
  sums.part = p.part;
  if (dnorm_in && !dy) ES_TRY(clear(dnorm_in, weight_dtype));  // no dy: zero, and no column sum
  ES_NORM_CALL(backward, p, sums, s);
  return ES_ERR_UNSUPPORTED;
}
