// fp8.hip — what writes the 8-bit format (fp8.h): a matrix quantised, the AdaLN normalisation quantised as it is
// written, and keys and values quantised into a cache. All three are bound by memory: every input element is read
// once (16 B a lane) and every code written once (8 B a lane).
//
// A lane holds 8 consecutive elements, so the 16 lanes of a DPP row hold one block of 128 (its amax is four row
// rotations away) and a wave holds four blocks: of a matrix row, one 32-bit word of scales.
#include "fp8.h"

namespace {

constexpr int MAXCH = 16;  // 512-column chunks of a row that a wave keeps in registers (AdaLN: dim <= 8192)

// this lane's 8 elements x (zeros past the row's end) -> its 8 codes; the block's scale byte
__device__ __forceinline__ uint32_t quant8(const float (&x)[8], uint2& codes) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, abs_bits(x[e]));
  const uint32_t b = e8m0_of(row16_max(m));
  const float r = e8m0_inv(b);
  codes = make_uint2(pack4_e4m3(x[0] * r, x[1] * r, x[2] * r, x[3] * r),
                     pack4_e4m3(x[4] * r, x[5] * r, x[6] * r, x[7] * r));
  return b;
}

// Waves of a launch, four a workgroup. A grid dimension holds fewer than 2^32 threads (a launch of more is cut without an
// error), so from 2^23 workgroups on they go to a second one.
constexpr int GRID_X = 23;
__device__ __forceinline__ int64_t wave_of_launch() {
  return (((int64_t)blockIdx.y << GRID_X) + blockIdx.x) * 4 + (threadIdx.x >> 6);
}
inline dim3 grid_of(int64_t waves) {
  const int64_t n = (waves + 3) / 4, x = min(n, (int64_t)1 << GRID_X);
  return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}

// the four blocks' bytes of a wave as one word (every lane); blocks from `nblk` on are 0
__device__ __forceinline__ uint32_t scale_word(uint32_t b, int nblk) {
  uint32_t w = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (g < nblk) w |= (uint32_t)__builtin_amdgcn_readlane((int)b, 16 * g) << (8 * g);
  return w;
}

// One wave per 512-column chunk (four blocks) of a row: no wave depends on another, so small matrices spread over the chip.
// 30720 x 2048 bf16: the kernel 32 us (5.9 TB/s), a call among others 36 (5.2; a copy's rate 4.9); 157 x 1360 fp32: 2.6 us.
template <typename T>
__global__ void __launch_bounds__(256) quantize_fp8_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols,
                                                           uint8_t* __restrict__ q, int64_t ldq,
                                                           uint32_t* __restrict__ scale, int64_t lds_) {
  const int lane = threadIdx.x & 63;
  const int chunks = (cols + 511) >> 9;
  const int64_t task = wave_of_launch();
  if (task >= (int64_t)rows * chunks) return;
  const int row = (int)(task / chunks), c = (int)(task - (int64_t)row * chunks);
  const int col = c * 512 + lane * 8;
  float v[8] = {};
  if (col < cols) load8(x + row * ldx + col, v);  // cols % 16 == 0
  uint2 codes;
  const uint32_t b = quant8(v, codes);
  if (col < cols) *(uint2*)(q + row * ldq + col) = codes;
  const uint32_t w = scale_word(b, (min(cols - c * 512, 512) + 127) >> 7);
  if (lane == 0) scale[c * lds_ + row] = w;
}

// y = (x * rsqrt(mean x^2 + eps)) * scale1 + shift in fp32, quantised: one wave per row, the row in registers, so that x is
// read once. CH: 512-column chunks held (2, 4, 8, 16 by dim). 30720 x 2048 bf16: the kernel 36 us (5.3 TB/s), a call
// among others 43 (4.4); 640 x 2048: 5.1 us, the latencies of a row's loads, its sum and the vectors' loads one after the other.
// Codes that differ from those of the 64-bit value: 62 to 77 of 63 million (as many as for torch's fp32 operations).
template <typename T, int CH>
__global__ void __launch_bounds__(256) adaln_fp8_kernel(const T* __restrict__ x, int rows, int dim,
                                                        const T* __restrict__ shift, const T* __restrict__ scale1,
                                                        int rows_per_vec, int64_t vec_stride, float eps,
                                                        uint8_t* __restrict__ q, int64_t ldq,
                                                        uint32_t* __restrict__ scale, int64_t lds_) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = wave_of_launch();
  if (wave >= rows) return;
  const int row = (int)wave;
  const T* xr = x + (int64_t)row * dim;
  float v[CH][8];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = c * 512 + lane * 8;
    if (col < dim) {
      load8(xr + col, v[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[c][e], v[c][e], ss);
  }
  ss = wave_sum(ss);
  const float r = 1.0f / sqrtf(ss / (float)dim + eps);
  const int64_t vo = (int64_t)(row / rows_per_vec) * vec_stride;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = c * 512 + lane * 8;
    if (c * 512 >= dim) break;
    if (col < dim) {
      float s1[8], sh[8];
      load8(scale1 + vo + col, s1);
      load8(shift + vo + col, sh);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = __builtin_fmaf(v[c][e] * r, s1[e], sh[e]);
    }
    uint2 codes;
    const uint32_t b = quant8(v[c], codes);
    if (col < dim) *(uint2*)(q + (int64_t)row * ldq + col) = codes;
    const uint32_t w = scale_word(b, (min(dim - c * 512, 512) + 127) >> 7);
    if (lane == 0) scale[c * lds_ + row] = w;
  }
}

// Keys and values of `nblk` layers into a cache: one wave per (token, layer, k | v, four heads), 16 lanes a head.
// Token t of sequence b goes to slot start[b] + t (start NULL: t) if t < lens[b] and the slot lies in the cache; every
// other slot keeps its bytes. Keys get the head RMS norm (w) and interleaved rotary pairs on heads < rope_heads, at
// position pos0 + pos_mult * slot; fp32 throughout, the only rounding is the code's.
// 2 x 1600 tokens (1800 of them valid), 24 layers, 16 heads, bf16: 182 us, 2.9 TB/s: the scale bytes of a
// token lie a capacity apart. 4 x 1: 3.5 us. Consecutive waves take consecutive bytes of x. Tokens in groups (2 to 16, so
// that their scale bytes, which lie beside each other, are written together) took 186 us, and an XCD's own range of tokens
// 250 us.
template <typename T>
__global__ void __launch_bounds__(256) kv_write_fp8_kernel(EchoKVWriteArgs a) {
  const int lane = threadIdx.x & 63;
  const int hg = (a.heads + 3) >> 2;
  const int64_t per = (int64_t)a.nblk * 2 * hg;
  const int64_t task = wave_of_launch();
  if (task >= (int64_t)a.batch * a.tokens * per) return;
  const int64_t row = task / per;
  int rest = (int)(task - row * per);
  const int g = rest % hg;
  rest /= hg;
  const int kv = rest & 1, blk = rest >> 1;
  const int b = (int)(row / a.tokens), t = (int)(row - (int64_t)b * a.tokens);
  if (a.lens && t >= a.lens[b]) return;
  const int64_t slot = (int64_t)t + (a.start ? a.start[b] : 0);
  if (slot < 0 || slot >= a.capacity) return;
  const int h = g * 4 + (lane >> 4), d0 = (lane & 15) * 8;
  const bool on = h < a.heads;
  float v[8] = {};
  if (on) load8((const T*)a.x + row * a.ldx + ((int64_t)(blk * 2 + kv) * a.heads + h) * 128 + d0, v);
  if (kv == 0) {
    if (a.w) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
      const float r = 1.0f / sqrtf(row16_sum(ss) / 128.0f + a.eps);
      float wv[8] = {};
      if (on) load8((const T*)a.w + ((int64_t)blk * a.heads + h) * 128 + d0, wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (v[e] * wv[e]) * r;  // v * w is exact for bf16
    }
    if (h < a.rope_heads) {
      const float* cs = a.rope + ((a.pos0 + a.pos_mult * slot) * 64 + d0 / 2) * 2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = cs[2 * e], s = cs[2 * e + 1], p = v[2 * e], o = v[2 * e + 1];
        v[2 * e] = __builtin_fmaf(p, c, -(o * s));
        v[2 * e + 1] = __builtin_fmaf(p, s, o * c);
      }
    }
  }
  uint2 codes;
  const uint32_t byte = quant8(v, codes);
  if (!on) return;
  *(uint2*)((uint8_t*)a.cache + b * a.c_batch + slot * a.c_tok + blk * a.c_blk + kv * a.c_kv + h * a.c_head + d0) = codes;
  if ((lane & 15) == 0)
    ((uint8_t*)a.scale)[b * a.s_batch + blk * a.s_blk + kv * a.s_kv + h * a.s_head + slot * a.s_tok] = (uint8_t)byte;
}

inline bool aligned(const void* p, int64_t ld, int bytes, int a = 16) {
  return (uintptr_t)p % a == 0 && (ld * bytes) % a == 0;
}

template <typename T, int CH>
void launch_adaln(const void* x, int rows, int dim, const void* shift, const void* scale1, int rpv, int64_t vs, float eps,
                  void* q, int64_t ldq, void* scale, int64_t lds_, hipStream_t st) {
  hipLaunchKernelGGL((adaln_fp8_kernel<T, CH>), grid_of(rows), dim3(256), 0, st, (const T*)x, rows, dim,
                     (const T*)shift, (const T*)scale1, rpv, vs, eps, (uint8_t*)q, ldq, (uint32_t*)scale, lds_);
}

template <typename T>
void launch_adaln_t(const void* x, int rows, int dim, const void* shift, const void* scale1, int rpv, int64_t vs,
                    float eps, void* q, int64_t ldq, void* scale, int64_t lds_, hipStream_t st) {
  const int ch = (dim + 511) / 512;
  if (ch <= 2) launch_adaln<T, 2>(x, rows, dim, shift, scale1, rpv, vs, eps, q, ldq, scale, lds_, st);
  else if (ch <= 4) launch_adaln<T, 4>(x, rows, dim, shift, scale1, rpv, vs, eps, q, ldq, scale, lds_, st);
  else if (ch <= 8) launch_adaln<T, 8>(x, rows, dim, shift, scale1, rpv, vs, eps, q, ldq, scale, lds_, st);
  else launch_adaln<T, MAXCH>(x, rows, dim, shift, scale1, rpv, vs, eps, q, ldq, scale, lds_, st);
}

}  // namespace

extern "C" {

int echo_quantize_fp8(int32_t dtype, const void* x, int64_t ldx, int32_t rows, int32_t cols, void* q, int64_t ldq,
                      void* scale, int64_t ld_scale, void* stream) {
  if (dtype != ECHO_BF16 && dtype != ECHO_F32) return ECHO_EDTYPE;
  if (rows < 0 || cols <= 0 || cols % 16 || ldx < cols || ldq < cols || ld_scale < rows) return ECHO_ESHAPE;
  if (rows == 0) return ECHO_OK;
  if (!x || !q || !scale) return ECHO_EINVAL;
  if (!aligned(x, ldx, dtype == ECHO_BF16 ? 2 : 4) || !aligned(q, ldq, 1) || (uintptr_t)scale % 4) return ECHO_EALIGN;
  const int64_t tasks = (int64_t)rows * ((cols + 511) / 512);
  if (tasks > (int64_t)4 * INT32_MAX) return ECHO_ESHAPE;
  const dim3 grid = grid_of(tasks);
  if (dtype == ECHO_BF16)
    hipLaunchKernelGGL(quantize_fp8_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16_t*)x, ldx, rows,
                       cols, (uint8_t*)q, ldq, (uint32_t*)scale, ld_scale);
  else
    hipLaunchKernelGGL(quantize_fp8_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)x, ldx, rows,
                       cols, (uint8_t*)q, ldq, (uint32_t*)scale, ld_scale);
  ECHO_LAUNCH_CHECK();
  return ECHO_OK;
}

int echo_adaln_modulate_fp8(int32_t dtype, const void* x, int32_t rows, int32_t dim, const void* shift,
                            const void* scale1, int32_t rows_per_vec, int64_t vec_stride, float eps, void* q,
                            int64_t ldq, void* scale, int64_t ld_scale, void* stream) {
  if (dtype != ECHO_BF16 && dtype != ECHO_F32) return ECHO_EDTYPE;
  if (rows < 0 || dim <= 0 || dim % 16 || dim > MAXCH * 512 || ldq < dim || ld_scale < rows) return ECHO_ESHAPE;
  if (rows == 0) return ECHO_OK;
  if (!x || !shift || !scale1 || !q || !scale) return ECHO_EINVAL;
  const int es = dtype == ECHO_BF16 ? 2 : 4;
  if (!aligned(x, dim, es) || !aligned(shift, vec_stride, es) || !aligned(scale1, vec_stride, es) || !aligned(q, ldq, 1) ||
      (uintptr_t)scale % 4)
    return ECHO_EALIGN;
  if (rows_per_vec <= 0) rows_per_vec = rows;
  if (dtype == ECHO_BF16)
    launch_adaln_t<bf16_t>(x, rows, dim, shift, scale1, rows_per_vec, vec_stride, eps, q, ldq, scale, ld_scale, (hipStream_t)stream);
  else
    launch_adaln_t<float>(x, rows, dim, shift, scale1, rows_per_vec, vec_stride, eps, q, ldq, scale, ld_scale, (hipStream_t)stream);
  ECHO_LAUNCH_CHECK();
  return ECHO_OK;
}

int echo_kv_write_fp8(const EchoKVWriteArgs* a, void* stream) {
  if (!a) return ECHO_EINVAL;
  if (a->dtype != ECHO_BF16 && a->dtype != ECHO_F32) return ECHO_EDTYPE;
  if (a->batch < 0 || a->tokens < 0 || a->capacity < 0 || a->nblk <= 0 || a->heads <= 0 ||
      a->ldx < (int64_t)a->nblk * 2 * a->heads * 128 || a->rope_heads < 0 || a->rope_heads > a->heads)
    return ECHO_ESHAPE;
  if (a->batch == 0 || a->tokens == 0 || a->capacity == 0) return ECHO_OK;
  if (!a->x || !a->cache || !a->scale || (a->rope_heads > 0 && !a->rope)) return ECHO_EINVAL;
  // every slot's position has to lie in the rotary table
  if (a->rope_heads > 0 && (a->pos0 < 0 || a->pos_mult < 0 ||
                            a->pos0 + (int64_t)a->pos_mult * (a->capacity - 1) >= a->rope_positions))
    return ECHO_ESHAPE;
  const int es = a->dtype == ECHO_BF16 ? 2 : 4;
  if (!aligned(a->x, a->ldx, es) || !aligned(a->cache, a->c_batch, 1, 8) || a->c_tok % 8 || a->c_blk % 8 || a->c_kv % 8 ||
      a->c_head % 8 || (a->w && (uintptr_t)a->w % 16))
    return ECHO_EALIGN;
  const int64_t tasks = (int64_t)a->batch * a->tokens * a->nblk * 2 * ((a->heads + 3) / 4);
  if (tasks > (int64_t)4 * INT32_MAX) return ECHO_ESHAPE;
  const dim3 grid = grid_of(tasks);
  if (a->dtype == ECHO_BF16)
    hipLaunchKernelGGL(kv_write_fp8_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, *a);
  else
    hipLaunchKernelGGL(kv_write_fp8_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, *a);
  ECHO_LAUNCH_CHECK();
  return ECHO_OK;
}

}  // extern "C"
