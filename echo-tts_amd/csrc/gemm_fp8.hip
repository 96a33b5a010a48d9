// gemm_fp8.hip — C[M,N] = tail(A[M,K] . W[N,K]^T) over the 8-bit format (fp8.h): e4m3 codes, one power-of-two scale for
// each block of 128 along K.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 rows over 128 of K, one block, and takes the scale of each
// row's block as an operand: the scaling costs no vector instruction, and one instruction stands for the two bf16
// MFMAs that 64 of K take in the same 32 cycles. The dot product does not care how K is permuted as long as both
// operands agree and the scale is one per 128, so lane group g reads the 16-B chunks g and g + 4 of a row: the LDS
// image is byte for byte that of the bf16 kernels (128 B a row, chunk ^ ((row >> 1) & 7), conflict-free).
// What the instruction adds in fixed point before fp32: products of 8 consecutive k, each cut toward zero to a multiple
// of 2^-13 of the largest one's power of two (measured by cancellation; about 2^-18 of sum |a w| on random inputs, the
// output's own rounding is 2^-9). The sums of the groups of 8 and over K are fp32.
// Operands are swapped (W fragment first) so that a lane ends with 4 consecutive output columns of one row.
// Tiles arrive by LDS-DMA with buffer addressing: rows past the matrix and the part of the last block past K read as
// zero codes. Scales of a tile (one word for 512 of K and row) are copied to LDS ahead of the K loop.
#include "fp8.h"

#include <type_traits>

extern int g_policy_num, g_policy_den;  // echo_set_policy_rows (gemm.hip)

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int BK = 128;       // bytes (= elements) of K per tile
constexpr int KSEG = 64;      // K-tiles whose scales are in LDS at a time (16 words a row)
constexpr uint32_t OOB = 0x80000000u;  // a byte offset past every buffer's range: reads as zero

// kinds of tail
enum { EK_STORE, EK_BIAS, EK_RESID, EK_RESID_BIAS, EK_SWIGLU, EK_SWIGLU_Q };
constexpr bool has_aux(int ek) { return ek == EK_RESID || ek == EK_RESID_BIAS; }
constexpr bool has_bias(int ek) { return ek == EK_BIAS || ek == EK_RESID_BIAS; }

// LDS-DMA of 16 B a lane from a buffer: LDS destination = lds_addr + lane * 16, out-of-range lanes get zeros
__device__ __forceinline__ void blds16(u32x4 rsrc, uint32_t voff, uint32_t lds_addr) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(rsrc), "s"(lds_addr) : "memory");
}

__device__ __forceinline__ u32x4 buffer_at(const uint8_t* p, int64_t bytes) {
  const uint64_t b = (uint64_t)p;
  const uint32_t n = bytes < 0 ? 0u : bytes > (int64_t)0x7ffffff0 ? 0x7ffffff0u : (uint32_t)bytes;
  u32x4 r;
  r[0] = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  r[1] = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(b >> 32) & 0xffffu));
  r[2] = (uint32_t)__builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000u;
  return r;
}

// 4 B a lane
__device__ __forceinline__ void blds4(u32x4 rsrc, uint32_t voff, uint32_t lds_addr) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(rsrc), "s"(lds_addr) : "memory");
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t out_buffer(void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)min(bytes, (int64_t)0x7ffffff0), 0x00020000);
}

template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int D>
__device__ __forceinline__ void vm_wait_stages(int n) {
  if (n >= 3) vm_wait<3 * D>();
  else if (n == 2) vm_wait<2 * D>();
  else if (n == 1) vm_wait<D>();
  else vm_wait<0>();
}


// silu(a) * b in fp32: the hardware reciprocal and exp2 (about 2 ulp) are far below the one rounding that follows. From
// a = -87 on down (FAR: where one may occur) the reciprocal of 1 + e^-a would leave the normal numbers; there 1 + e^a is 1,
// and e^a goes to both factors by halves, (a e^(a/2)) (b e^(a/2)): down to a = -174 no half underflows where the product
// does not
constexpr float SILU_FAR = -87.0f;
template <bool FAR = true>
__device__ __forceinline__ float swiglu_f(float a, float b) {
  const bool far = FAR && a < SILU_FAR;
  const float e = __builtin_amdgcn_exp2f(a * (far ? 0.72134752044448170f : -1.44269504088896341f));
  return FAR ? (a * (far ? e : __builtin_amdgcn_rcpf(1.0f + e))) * (far ? b * e : b) : a * __builtin_amdgcn_rcpf(1.0f + e) * b;
}

__device__ __forceinline__ void load4(const bf16_t* p, float (&o)[4]) {
  const uint2 u = *(const uint2*)p;
  o[0] = bf2f(u.x & 0xffffu); o[1] = bf2f(u.x >> 16); o[2] = bf2f(u.y & 0xffffu); o[3] = bf2f(u.y >> 16);
}
__device__ __forceinline__ void store4(bf16_t* p, const float (&v)[4]) {
  *(uint2*)p = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
}

// Output tail of one wave's TM x TN accumulators, from registers: lane holds row (lane & 15) of each 16-row fragment and
// 4 consecutive columns 4 (lane >> 4) .. + 3 of each 16-column fragment. EK_SWIGLU_Q: the 256 W rows of a tile are one
// 128-column block of every output row; its amax crosses the waves through xmax [WN][BM].
template <int BM, int BN, int WN, int FM, int FN, int EK>
__device__ __forceinline__ void fp8_tail(f32x4 (&acc)[FM][FN], int m0, int n0, int wm, int wn, int lane,
                                         const EchoGemmFp8Args& a, uint32_t* xmax) {
  constexpr int TM = FM * 16, TN = FN * 16;
  const int r16 = lane & 15, g = lane >> 4;
  if constexpr (EK == EK_STORE || EK == EK_BIAS || has_aux(EK)) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn * TN + j * 16 + 4 * g;
      if (n >= a.N) continue;
      float b[4] = {0.f, 0.f, 0.f, 0.f}, gt[4] = {1.f, 1.f, 1.f, 1.f};
      if (has_bias(EK)) load4((const bf16_t*)a.bias + n, b);
      if (has_aux(EK) && a.gate) load4((const bf16_t*)a.gate + n, gt);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = m0 + wm * TM + i * 16 + r16;
        if (m >= a.M) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] + b[e];
        if constexpr (has_aux(EK)) {
          float x[4];
          load4((const bf16_t*)a.aux + (int64_t)m * a.ld_aux + n, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(gt[e], v[e], x[e]);
        }
        store4((bf16_t*)a.C + (int64_t)m * a.ldc + n, v);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int p = 0; p < FN / 2; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][2 * p][e] = swiglu_f(acc[i][2 * p][e], acc[i][2 * p + 1][e]);
    const int c0 = (n0 + wn * TN) / 2 + 4 * g;  // output column of fragment pair 0
    if constexpr (EK == EK_SWIGLU) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = m0 + wm * TM + i * 16 + r16;
#pragma unroll
        for (int p = 0; p < FN / 2; ++p) {
          const float v[4] = {acc[i][2 * p][0], acc[i][2 * p][1], acc[i][2 * p][2], acc[i][2 * p][3]};
          if (m < a.M && c0 + p * 16 < a.N / 2) store4((bf16_t*)a.C + (int64_t)m * a.ldc + c0 + p * 16, v);
        }
      }
    } else {
      static_assert(BN == 256, "one 128-column output block a tile");
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        uint32_t mx = 0;
#pragma unroll
        for (int p = 0; p < FN / 2; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = max(mx, c0 + p * 16 < a.N / 2 ? abs_bits(acc[i][2 * p][e]) : 0u);
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
        if (g == 0) xmax[wn * BM + wm * TM + i * 16 + r16] = mx;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int ml = wm * TM + i * 16 + r16, m = m0 + ml;
        uint32_t mx = xmax[ml];
#pragma unroll
        for (int w = 1; w < WN; ++w) mx = max(mx, xmax[w * BM + ml]);
        const uint32_t b = e8m0_of(mx);
        const float r = e8m0_inv(b);
        if (m >= a.M) continue;
#pragma unroll
        for (int p = 0; p < FN / 2; ++p)
          if (c0 + p * 16 < a.N / 2)
            *(uint32_t*)((uint8_t*)a.C + (int64_t)m * a.ldc + c0 + p * 16) =
                pack4_e4m3(acc[i][2 * p][0] * r, acc[i][2 * p][1] * r, acc[i][2 * p][2] * r, acc[i][2 * p][3] * r);
        const int blk = n0 >> 8;  // output block; behind the last one the word's bytes are 0
        if (wn == 0 && g == 0) {
          uint8_t* sp = (uint8_t*)a.c_scale + ((int64_t)(blk >> 2) * a.ld_cs + m) * 4;
          sp[blk & 3] = (uint8_t)b;
          if (n0 + 256 >= a.N)
            for (int z = (blk & 3) + 1; z < 4; ++z) sp[z] = 0;
        }
      }
    }
  }
}

// tile -> block: XCD-chunked, then columns of up to GM row tiles (W and A tiles re-used from an XCD's L2)
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int GM, int& tm, int& tn) {
  const int nwg = tiles_m * tiles_n;
  const int xcd = bid & 7, q8 = nwg >> 3, r8 = nwg & 7;
  const int wg = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (bid >> 3);
  const int grp = wg / (GM * tiles_n);
  const int fm = grp * GM;
  const int gm = min(tiles_m - fm, GM);
  const int rem = wg - grp * GM * tiles_n;
  tm = fm + rem % gm;
  tn = rem / gm;
}

// WM x WN waves on a BM x BN tile, an NS-stage LDS ring with NS - 1 K-tiles in flight.
template <int BM, int BN, int WM, int WN, int NS, int EK>
__global__ void __launch_bounds__(64 * WM * WN)
gemm_fp8_ring_kernel(EchoGemmFp8Args a, int tiles_m, int tiles_n) {
  constexpr int NW = WM * WN, NT = 64 * NW;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int STAGE = (BM + BN) * BK;
  constexpr int AI = BM * 8 / NT, BI = BN * 8 / NT;  // DMA instructions per wave and K-tile (8 rows each)
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole DMA instructions");
  static_assert((AI + BI) * (NS - 2) <= 63, "vmcnt range");
  __shared__ __attribute__((aligned(16))) uint8_t lds[NS * STAGE];
  __shared__ uint32_t scl[KSEG / 4][BM + BN];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / WN, wn = wid % WN;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int nkt = (a.K + BK - 1) / BK;
  const uint8_t* Ab = (const uint8_t*)a.A + (int64_t)m0 * a.lda;
  const uint8_t* Wb = (const uint8_t*)a.W + (int64_t)n0 * a.ldw;
  const int64_t abytes = (int64_t)(a.M - 1 - m0) * a.lda + a.K, wbytes = (int64_t)(a.N - 1 - n0) * a.ldw + a.K;

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto stage = [&](int kt, int slot) __attribute__((always_inline)) {
    const int64_t k0 = (int64_t)kt * BK;
    const u32x4 ra = buffer_at(Ab + k0, abytes - k0), rw = buffer_at(Wb + k0, wbytes - k0);
    const int left = a.K - (int)k0;  // bytes of this K-tile inside the matrices
    const uint32_t dst = lds_addr_of(lds) + (uint32_t)slot * STAGE;
#pragma unroll
    for (int i = 0; i < AI + BI; ++i) {
      const bool isA = i < AI;
      const int rb = ((isA ? i : i - AI) * NW + wid) * 8;
      const int row = rb + (lane >> 3);
      const int c = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
      const uint32_t off = c < left ? (uint32_t)(row * (int)(isA ? a.lda : a.ldw) + c) : OOB;
      blds16(isA ? ra : rw, off, __builtin_amdgcn_readfirstlane(dst + (isA ? 0 : BM * BK) + rb * BK));
    }
  };
  const int frow = lane & 15, fsw = frow >> 1, g = lane >> 4;
  auto frag = [&](const uint8_t* tile, int row) __attribute__((always_inline)) {
    const i32x4 lo = *(const i32x4*)(tile + row * BK + ((g ^ fsw) * 16));
    const i32x4 hi = *(const i32x4*)(tile + row * BK + (((g + 4) ^ fsw) * 16));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  for (int s0 = 0; s0 < nkt; s0 += KSEG) {  // K beyond 8192: the ring drains, the next scales are loaded
    const int nk = min(nkt - s0, KSEG), q0 = s0 >> 2, nq = (nk + 3) >> 2;
    if (s0 != 0) __syncthreads();
#pragma unroll
    for (int p = 0; p < NS - 1; ++p)
      if (p < nk) stage(s0 + p, p);
    for (int x = tid; x < nq * (BM + BN); x += NT) {
      const int q = x / (BM + BN), r = x - q * (BM + BN);
      scl[q][r] = r < BM ? ((const uint32_t*)a.a_scale)[(int64_t)(q0 + q) * a.ld_as + min(m0 + r, a.M - 1)]
                         : ((const uint32_t*)a.w_scale)[(int64_t)(q0 + q) * a.ld_ws + min(n0 + r - BM, a.N - 1)];
    }
    for (int kt = 0; kt < nk; ++kt) {
      // this wave's share of K-tile kt has landed (the younger ones stay in flight), then everybody's; every wave is
      // done reading the slot that K-tile kt + NS - 1 goes to
      vm_wait_stages<AI + BI>(min(NS - 2, nk - 1 - kt));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      if (kt + NS - 1 < nk) stage(s0 + kt + NS - 1, (kt + NS - 1) % NS);
      const uint8_t* At = lds + (kt % NS) * STAGE;
      const uint8_t* Wt = At + BM * BK;
      const int q = kt >> 2, sh = (kt & 3) * 8;
      i32x8 xf[FM], wf[FN];
      uint32_t xs[FM], wsc[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        xf[i] = frag(At, wm * TM + i * 16 + frow);
        xs[i] = scl[q][wm * TM + i * 16 + frow] >> sh;
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        wf[j] = frag(Wt, wn * TN + j * 16 + frow);
        wsc[j] = scl[q][BM + wn * TN + j * 16 + frow] >> sh;
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf[i], acc[i][j], 0, 0, 0, wsc[j], 0, xs[i]);
    }
  }
  __syncthreads();  // xmax re-uses the stages
  fp8_tail<BM, BN, WN, FM, FN, EK>(acc, m0, n0, wm, wn, lane, a, (uint32_t*)lds);
}

// ------------------------------------------------------------------------------------------------ few tiles
// Launches that do not fill the chip are bound by latency and by the bytes in flight, not by MFMA: the KW waves of a
// workgroup share K (wave -> K-tiles w, w + KW, ..), each with an LDS ring of its own (NS stages, NS - 1 K-tiles in flight)
// that no barrier guards. (Fragments straight from memory cost four times the L1 cycles: the lanes of a fragment's four
// neighbours are four rows.) The parts are joined in LDS once, in a fixed order; the tail's waves take 2 column fragments.
template <int FM, int FN, int KW, int NS, int EK>
__global__ void __launch_bounds__(64 * KW)
gemm_fp8_few_kernel(EchoGemmFp8Args a, int tiles_m, int tiles_n) {
  constexpr int BM = FM * 16, BN = FN * 16, RI = (FM + FN) * 2, DI = RI + 2;  // DMA instructions a K-tile: rows, + scales
  constexpr int STAGE = (FM + FN) * 2048 + 512;  // [A rows | W rows][128 B], then the scale words of 64 + 64 rows
  constexpr int FNT = FN == 1 ? 1 : 2, WNT = FN / FNT, FMT = (FM * WNT + KW - 1) / KW, WMT = FM / FMT;
  static_assert(FM <= 4 && FN <= 4 && FM % FMT == 0 && WNT * WMT <= KW && DI * (NS - 1) <= 63, "few tiles");
  constexpr int RING = KW * NS * STAGE, PARTS = KW * FM * FN * 1024;
  __shared__ __attribute__((aligned(16))) uint8_t lds[RING > PARTS ? RING : PARTS];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int nkt = (a.K + BK - 1) / BK, mine = nkt > w ? (nkt - w + KW - 1) / KW : 0;
  const uint8_t* const Ab = (const uint8_t*)a.A + (int64_t)m0 * a.lda;
  const uint8_t* const Wb = (const uint8_t*)a.W + (int64_t)n0 * a.ldw;
  const int64_t abytes = (int64_t)(a.M - 1 - m0) * a.lda + a.K, wbytes = (int64_t)(a.N - 1 - n0) * a.ldw + a.K;
  uint8_t* const ring = lds + w * NS * STAGE;
  const uint32_t ring0 = __builtin_amdgcn_readfirstlane(lds_addr_of(lds)) + (uint32_t)(w * NS * STAGE);

  auto stage = [&](int x, int slot) __attribute__((always_inline)) {  // this wave's K-tile x
    const int kt = w + x * KW, left = a.K - kt * BK;
    const int64_t k0 = (int64_t)kt * BK;
    const u32x4 ra = buffer_at(Ab + k0, abytes - k0), rw = buffer_at(Wb + k0, wbytes - k0);
    const uint32_t dst = ring0 + (uint32_t)slot * STAGE;
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const bool isA = i < FM * 2;
      const int rb = (isA ? i : i - FM * 2) * 8, row = rb + (lane >> 3);
      const int c = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
      blds16(isA ? ra : rw, c < left ? (uint32_t)(row * (int)(isA ? a.lda : a.ldw) + c) : OOB, dst + (uint32_t)i * 1024);
    }
    const int64_t q = kt >> 2;
    blds4(buffer_at((const uint8_t*)a.a_scale + (q * a.ld_as + m0) * 4, (int64_t)(a.M - m0) * 4), (uint32_t)lane * 4, dst + (FM + FN) * 2048);
    blds4(buffer_at((const uint8_t*)a.w_scale + (q * a.ld_ws + n0) * 4, (int64_t)(a.N - n0) * 4), (uint32_t)lane * 4, dst + (FM + FN) * 2048 + 256);
  };
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < NS - 1; ++p)
    if (p < mine) stage(p, p);
  for (int x = 0; x < mine; ++x) {
    vm_wait_stages<DI>(min(NS - 2, mine - 1 - x));
    if (x + NS - 1 < mine) stage(x + NS - 1, (x + NS - 1) % NS);  // the slot of K-tile x - 1, whose reads are done
    const uint8_t* const T = ring + (x % NS) * STAGE;
    const int sh = w + x * KW;
    i32x8 fr[FM + FN];
    uint32_t sc[FM + FN];
#pragma unroll
    for (int f = 0; f < FM + FN; ++f) {
      const uint8_t* const row = T + (f * 16 + r16) * BK;
      const i32x4 lo = *(const i32x4*)(row + ((g ^ (r16 >> 1)) * 16)), hi = *(const i32x4*)(row + (((g + 4) ^ (r16 >> 1)) * 16));
      fr[f] = i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      sc[f] = T[(FM + FN) * 2048 + (f < FM ? f * 64 : 256 + (f - FM) * 64) + r16 * 4 + (sh & 3)];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fr[FM + j], fr[i], acc[i][j], 0, 0, 0, sc[FM + j], 0, sc[i]);
  }

  // parts [wave][fragment][lane], over the rings
  __syncthreads();
  f32x4* const part = (f32x4*)lds;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) part[((w * FM + i) * FN + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (w >= WNT * WMT) return;
  const int wn = w % WNT, wm = w / WNT;
  f32x4 sum[FMT][FNT];
#pragma unroll
  for (int i = 0; i < FMT; ++i)
#pragma unroll
    for (int j = 0; j < FNT; ++j) {
      const f32x4* const p = part + ((wm * FMT + i) * FN + wn * FNT + j) * 64 + lane;
      sum[i][j] = p[0];
#pragma unroll
      for (int k = 1; k < KW; ++k) sum[i][j] += p[k * FM * FN * 64];
    }
  fp8_tail<BM, BN, WNT, FMT, FNT, EK>(sum, m0, n0, wm, wn, lane, a, nullptr);
}

// ------------------------------------------------------------------------------------------------ many tiles
// Persistent 256 x 256 tiles for launches that fill the chip: one workgroup of 4 waves (2 x 2) a CU, one wave a SIMD with
// the whole register file: 128 x 128 outputs a wave (256 accumulators, v_mfma_scale_f32_32x32x64_f8f6f4). Against 8 waves
// of 128 x 64 this reads 2/3 of the LDS bytes per MFMA. A block of K (128) is computed in two steps of 16 MFMAs (64 cycles
// each): the wave's A rows 0-63 (A1), then 64-127 (A2), against its W fragments, which stay in registers for both. Between
// the MFMAs, in order:
//   step 0 of block b: the fragment reads of A2(b) (8), and the LDS-DMA of W and A1 of block b + 2 (12 instructions)
//   step 1 of block b: the fragment reads of W and A1 of block b + 1 (24), and the LDS-DMA of A2(b + 2) (4)
// so two LDS slots of a block do: what a step requests goes where everything was read a step before, and has two to three
// steps to land. A DMA instruction takes 8 whole rows of 128 B: at 64 B a row (steps of half a block, four slots) L2 serves
// one request a clock and channel at half width and was the bound (30720x8192x2048: 485 us, 66 % of the cycles in MFMA;
// now 424 us on one input, 436 on new inputs each time, 2.4 PFLOP/s at the clock that the card's power limit leaves;
// 30720x11776x2048 SwiGLU to 8 bits 604 and 630).
// One barrier a step: at its start every wave has its fragments in registers and everybody's share of what the step reads
// has landed (vmcnt counts in issue order: 16 younger operations stay in flight, whichever step it is).
// After a tile's last step the next tile's two blocks are requested before the epilogue, which works from the
// accumulators. A wave issues SN stores a tile (pieces outside the matrix go to an offset that the buffer drops), and the
// first three steps of the next tile leave them in flight.
constexpr int PS_KQ = 15;  // words of scales a row: K <= 7680
constexpr int PS_SLOT = 512 * BK;
constexpr int ps_stores(int ek) { return ek == EK_SWIGLU ? 16 : ek == EK_SWIGLU_Q ? 9 : 32; }

template <int EK>
__global__ void __launch_bounds__(256, 1) gemm_fp8_ps_kernel(EchoGemmFp8Args a, int tiles_m, int tiles_n, int group_m) {
  constexpr int BM = 256, BN = 256, SN = ps_stores(EK);
  // [2 slots][A 256 rows | W 256 rows][128 B], the 16-B chunk c of row r at c ^ ((r >> 1) & 7): conflict-free for the
  // fragment reads of 16 consecutive rows; then the scale words [PS_KQ][A 256 | W 256], the row maxima [2][256]
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * PS_SLOT + PS_KQ * 2048 + 2048];
  uint32_t* const xmax = (uint32_t*)(lds + 2 * PS_SLOT + PS_KQ * 2048);

  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int ntl = tiles_m * tiles_n;
  const int nb2 = a.K / BK, nq = (nb2 + 3) >> 2, nbe = (nb2 + 1) & ~1;  // blocks of K: K % 128 == 0, K >= 384 (host)
  const int nout = EK == EK_SWIGLU || EK == EK_SWIGLU_Q ? a.N / 2 : a.N;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr_of(lds));

  // Every address starts from an opaque copy of the lane: what lives from tile to tile would be spilled, and a reload waits
  // for all DMA in flight.
  auto opaque = [&]() __attribute__((always_inline)) {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
  };
  // this lane's place in the wave's first DMA rows (8 rows x 8 chunks, swizzled at the source: rows 8 x .. have their chunk
  // bit 2 flipped for odd x). A: rows (wid >> 1) * 128 + (wid & 1) * 32 + 8 x (A1; A2 64 below), W: wid * 64 + 8 x
  uint32_t da[2], dw[2];
  auto offsets = [&]() __attribute__((always_inline)) {
    const int l = opaque(), ra = (wid >> 1) * 128 + (wid & 1) * 32 + (l >> 3), rw = wid * 64 + (l >> 3);
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int c = ((l & 7) ^ (l >> 4) ^ (4 * o)) * 16;
      da[o] = (uint32_t)(ra * (int)a.lda + c);
      dw[o] = (uint32_t)(rw * (int)a.ldw + c);
    }
  };
  int m0, n0;
  // buffers at the tile's rows and the block to request. Their range stays that of block 0 as the base moves on: a row past
  // the matrix has an offset behind it in any case (ld >= K), and K is whole
  u32x4 ra, rw;
  auto aim = [&]() __attribute__((always_inline)) {
    ra = buffer_at((const uint8_t*)a.A + m0 * a.lda, (a.M - 1 - m0) * a.lda + a.K);
    rw = buffer_at((const uint8_t*)a.W + n0 * a.ldw, (a.N - 1 - n0) * a.ldw + a.K);
  };
  auto advance = [&](u32x4& r, uint32_t by) __attribute__((always_inline)) {
    const uint64_t x = (((uint64_t)r[1] << 32) | r[0]) + by;
    r[0] = (uint32_t)x;
    r[1] = (uint32_t)(x >> 32);
  };
  auto slot_at = [&](int b) __attribute__((always_inline)) {
    uint32_t x = lds0 + (uint32_t)(b & 1) * PS_SLOT;
    asm volatile("" : "+s"(x));  // or the pieces' addresses of both slots are held (and spilled)
    return x;
  };
  // x: 0-7 W, 8-11 A1, 12-15 A2
  auto piece = [&](int x, uint32_t slot) __attribute__((always_inline)) {
    if (x < 8) {
      blds16(rw, dw[x & 1] + (uint32_t)(8 * x * (int)a.ldw), slot + 32768 + wid * 8192 + x * 1024);
    } else {
      const int row = (x & 3) * 8 + (x < 12 ? 0 : 64);
      blds16(ra, da[x & 1] + (uint32_t)(row * (int)a.lda), slot + (wid >> 1) * 16384 + (wid & 1) * 4096 + row * BK);
    }
  };
  // scales (128 words a wave and word row: waves 0, 1 the A rows, 2, 3 the W rows), then blocks 0 and 1
  auto prologue = [&]() __attribute__((always_inline)) {
    const int64_t r0 = wid < 2 ? m0 : n0, rows = wid < 2 ? a.M : a.N;
    const uint32_t* sp = (const uint32_t*)(wid < 2 ? a.a_scale : a.w_scale) + r0;
    const int64_t ls = wid < 2 ? a.ld_as : a.ld_ws;
    for (int q = 0; q < nq; ++q) {
      const u32x4 r = buffer_at((const uint8_t*)(sp + q * ls), (rows - r0) * 4);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        blds4(r, (uint32_t)(((wid & 1) * 128 + h * 64 + opaque()) * 4), lds0 + (uint32_t)(2 * PS_SLOT + q * 2048 + wid * 512 + h * 256));
    }
    offsets();
    aim();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b) { advance(ra, BK); advance(rw, BK); }
#pragma unroll
      for (int x = 0; x < 16; ++x) piece(x, lds0 + b * PS_SLOT);
    }
  };
  auto origin = [&](int t) __attribute__((always_inline)) {
    int tm, tn;
    tile_of(t, tiles_m, tiles_n, group_m, tm, tn);
    m0 = tm * BM;
    n0 = tn * BN;
  };

  int t = blockIdx.x;
  if (t >= ntl) return;
  origin(t);
  prologue();
  bool first = true;
  for (;;) {
    f32x16 acc[4][4];
    // fragments of 32 rows: [half of K][chunk]; lane l holds row l & 31, chunks 4 h + (l >> 5) and + 2 of half h
    i32x4 fa[4][2][2], fw[2][4][2][2];
    uint32_t as[4], ws[4], an[4], wn_[4];
    // the lane's row in slot 0 and its scale words; the rest is immediate
    const int kl = opaque();
    const uint32_t fr = (uint32_t)((kl & 31) * BK + (((kl >> 5) ^ ((kl >> 1) & 7)) * 16));
    const uint32_t fra = fr + wm * 16384, frw = fr + 32768 + wn * 16384;
    const uint32_t sca = (uint32_t)(2 * PS_SLOT + (wm * 128 + (kl & 31)) * 4), scw = (uint32_t)(2 * PS_SLOT + 1024 + (wn * 128 + (kl & 31)) * 4);
    offsets();
    uint32_t pa, pw;
    // x: chunk x & 1 of half (x >> 1) & 1 of fragment x >> 2
    auto read_a = [&](int x) __attribute__((always_inline)) {
      fa[x >> 2][(x >> 1) & 1][x & 1] = *(const i32x4*)(lds + (pa ^ ((x & 3) * 32)) + (x >> 2) * 4096);
    };
    auto read_w = [&](int set, int x) __attribute__((always_inline)) {
      // halves of K are chunk bit 2 (64 B), the lane's second chunk is bit 1 (32 B)
      fw[set][x >> 2][(x >> 1) & 1][x & 1] = *(const i32x4*)(lds + (pw ^ ((x & 3) * 32)) + (x >> 2) * 4096);
    };
    auto scales = [&](int blk) __attribute__((always_inline)) {
      uint32_t o = (uint32_t)((blk >> 2) * 2048 + (blk & 3));
      asm volatile("" : "+s"(o));
      const uint32_t qa = sca + o, qw = scw + o;
#pragma unroll
      for (int f = 0; f < 4; ++f) { an[f] = lds[qa + f * 128]; wn_[f] = lds[qw + f * 128]; }
    };
    // step H of a block with W set S. RD: its reads (H 0: A2 of this block, H 1: W (set 1 - S) and A1 of the next);
    // DM: its requests into `slot`; Z: the tile's first block (the accumulators start from the instruction's zero)
    auto step = [&](auto hh, auto ss, auto rd, auto dm, uint32_t slot, auto z) __attribute__((always_inline)) {
      constexpr int H = decltype(hh)::value, S = decltype(ss)::value;
#pragma unroll
      for (int m = 0; m < 16; ++m) {
        const int kh = m >> 3, i = 2 * H + ((m >> 2) & 1), j = (m & 4) ? 3 - (m & 3) : (m & 3);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            __builtin_shufflevector(fw[S][j][kh][0], fw[S][j][kh][1], 0, 1, 2, 3, 4, 5, 6, 7),
            __builtin_shufflevector(fa[i][kh][0], fa[i][kh][1], 0, 1, 2, 3, 4, 5, 6, 7),
            decltype(z)::value && kh == 0 ? f32x16{} : acc[i][j], 0, 0, 0, ws[j], 0, as[i]);
        if constexpr (decltype(rd)::value) {
          if (H == 0) {
            if (m < 8) read_a(8 + m);
          } else {
            read_w(1 - S, m);
            if (m & 1) read_a(m >> 1);
          }
        }
        if constexpr (decltype(dm)::value) {
          if (H == 0) {
            if (m >= 4) piece(m - 4, slot);
          } else {
            if (m >= 2 && m < 6) piece(10 + m, slot);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // pinned here (no instruction): or the compiler sinks a step's MFMAs behind the next one's reads
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+a"(acc[2 * H + i][j]));
    };
    auto meet = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    using Y = std::true_type;
    using N = std::false_type;
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    auto look = [&](int b) __attribute__((always_inline)) {  // block b is read from here
      uint32_t o = (uint32_t)(b & 1) * PS_SLOT;
      asm volatile("" : "+s"(o));
      pa = fra + o;
      pw = frw + o;
    };
    auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int f = 0; f < 4; ++f) { as[f] = an[f]; ws[f] = wn_[f]; }
    };
    // block b with W set S, W0 / W1 operations still in flight at the starts of its steps. No branch inside.
    auto block = [&](int b, auto ss, auto w0, auto w1, auto z) __attribute__((always_inline)) {
      take_scales();
      vm_wait<decltype(w0)::value>();
      meet();
      advance(ra, b + 2 < nb2 ? BK : 0);
      advance(rw, b + 2 < nb2 ? BK : 0);
      const uint32_t slot = slot_at(b);
      step(I0{}, ss, Y{}, Y{}, slot, z);
      vm_wait<decltype(w1)::value>();
      meet();
      look(b + 1);
      scales(b + 1);
      step(I1{}, ss, Y{}, Y{}, slot, z);
    };
    using W = std::integral_constant<int, 16>;
    using WS = std::integral_constant<int, 16 + SN>;  // the previous tile's stores still count
    // the first tile of a workgroup has no stores to leave in flight: it waits for both blocks
    if (first) vm_wait<0>(); else vm_wait<20 + SN>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    look(0);
    scales(0);
#pragma unroll
    for (int x = 0; x < 16; ++x) read_w(0, x);
#pragma unroll
    for (int x = 0; x < 8; ++x) read_a(x);
    // the W sets alternate from block to block, so the blocks go in pairs; an odd number of them is filled up with the last
    // one once more, its scales 0 (2^-127 each: every product underflows, and what is NaN there is NaN in its row already)
    block(0, I0{}, WS{}, WS{}, Y{});
    block(1, I1{}, WS{}, W{}, N{});
#pragma unroll 1
    for (int b = 2; b < nbe - 2; b += 2) {
      block(b, I0{}, W{}, W{}, N{});
      block(b + 1, I1{}, W{}, W{}, N{});
    }
    // the last two request nothing
    take_scales();
    vm_wait<16>();
    meet();
    step(I0{}, I0{}, Y{}, N{}, 0, N{});
    vm_wait<4>();
    meet();
    look(nbe - 1);
    scales(nb2 - 1);
    step(I1{}, I0{}, Y{}, N{}, 0, N{});
    take_scales();
    const uint32_t keep = nbe == nb2 ? 255 : 0;
#pragma unroll
    for (int f = 0; f < 4; ++f) as[f] &= keep;
#pragma unroll
    for (int f = 0; f < 4; ++f) ws[f] &= keep;
    vm_wait<0>();
    meet();
    step(I0{}, I1{}, Y{}, N{}, 0, N{});
    meet();  // every wave has its last fragments: the slots and the scales are free
    step(I1{}, I1{}, N{}, N{}, 0, N{});

    // ---- epilogue. acc[i][j][4 q + e]: row wm * 128 + 32 i + r32, column wn * 128 + 32 j + 8 q + 4 g2 + e.
    // v_permlane32_swap of two quads' packed words leaves lanes 0-31 with 8 consecutive columns of the first and lanes
    // 32-63 of the second; v_permlane16_swap of two such pieces then turns 32 rows x 32 B into 16 rows x 64 B.
    constexpr int es = EK == EK_SWIGLU_Q ? 1 : 2;
    const int64_t m0c = m0;
    const int n0c = n0;
    const int el = opaque();
    const int r32 = el & 31, g2 = el >> 5, l16 = el & 15, g16 = el >> 4;
    const __amdgpu_buffer_rsrc_t crs = out_buffer((uint8_t*)a.C + m0c * a.ldc * es, ((a.M - 1 - m0c) * a.ldc + nout) * es);
    const int tnext = t + gridDim.x;
    const bool more = tnext < ntl;
    // rows x 64 B pieces: y = 0 / 1 the fragment's rows 0-15 / 16-31; byte column cb of this lane's 16
    auto put = [&](u32x4 p, u32x4 q, int i, int cb, bool in) __attribute__((always_inline)) {
      u32x4 lo, hi;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const auto s = __builtin_amdgcn_permlane16_swap(p[w], q[w], false, false);
        lo[w] = s[0];
        hi[w] = s[1];
      }
      const uint32_t off = (uint32_t)((wm * 128 + i * 32 + l16) * a.ldc * es) + cb;
      __builtin_amdgcn_raw_buffer_store_b128(lo, crs, in ? off : OOB, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(hi, crs, in ? off + (uint32_t)(16 * a.ldc * es) : OOB, 0, 0);
      __builtin_amdgcn_sched_barrier(0);  // one piece at a time: or all 256 accumulators are read at once, and spill
    };
    if constexpr (EK == EK_STORE || EK == EK_BIAS || has_aux(EK)) {
      // lane's columns of piece (j, k) (16 columns 32 j + 16 k of the wave's 128) before the row exchange
      const int cw = n0c + wn * 128 + 8 * g2;
      u32x4 bs[8], gt[8], xr[2][8];  // bf16 pairs; the residual rows of two fragments in flight
      // no branch: columns past N and a missing vector lie outside the buffer and read as 0
      const __amdgpu_buffer_rsrc_t brs = out_buffer(const_cast<void*>(a.bias), a.bias ? (int64_t)a.N * 2 : 0);
      const __amdgpu_buffer_rsrc_t grs = out_buffer(const_cast<void*>(a.gate), a.gate ? (int64_t)a.N * 2 : 0);
      const uint32_t one = a.gate ? 0u : 0x3f803f80u;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if constexpr (has_bias(EK))
          bs[p] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(brs, (uint32_t)((cw + p * 16) * 2), 0, 0));
        if constexpr (has_aux(EK)) {
          gt[p] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(grs, (uint32_t)((cw + p * 16) * 2), 0, 0));
          gt[p] |= u32x4{one, one, one, one};
        }
      }
      auto rows = [&](int i) __attribute__((always_inline)) {
        if constexpr (has_aux(EK)) {
          const __amdgpu_buffer_rsrc_t ars =
              out_buffer((uint8_t*)const_cast<void*>(a.aux) + m0c * a.ld_aux * 2, ((a.M - 1 - m0c) * a.ld_aux + a.N) * 2);
#pragma unroll
          for (int p = 0; p < 8; ++p)
            xr[i & 1][p] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                ars, cw + p * 16 < a.N ? (uint32_t)(((wm * 128 + i * 32 + r32) * a.ld_aux + cw + p * 16) * 2) : OOB, 0, 0));
        }
      };
      rows(0);
      rows(1);
      if (more) {
        origin(tnext);
        prologue();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          asm volatile("" : "+a"(acc[i][j]));  // read from here on, not ahead
          u32x4 o[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if constexpr (EK == EK_STORE) {
              const f32x16& u = acc[i][j];
              const auto x = __builtin_amdgcn_permlane32_swap(pack2bf(u[8 * k], u[8 * k + 1]), pack2bf(u[8 * k + 4], u[8 * k + 5]), false, false);
              const auto y = __builtin_amdgcn_permlane32_swap(pack2bf(u[8 * k + 2], u[8 * k + 3]), pack2bf(u[8 * k + 6], u[8 * k + 7]), false, false);
              o[k] = u32x4{x[0], y[0], x[1], y[1]};
              continue;
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][8 * k + e]),
                                                              __float_as_uint(acc[i][j][8 * k + 4 + e]), false, false);
              v[e] = __uint_as_float(s[0]);
              v[4 + e] = __uint_as_float(s[1]);
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (has_bias(EK)) {
                v[2 * w] += bf2f(bs[2 * j + k][w] & 0xffffu);
                v[2 * w + 1] += bf2f(bs[2 * j + k][w] >> 16);
              }
              if constexpr (has_aux(EK)) {
                const uint32_t x = xr[i & 1][2 * j + k][w], g = gt[2 * j + k][w];
                v[2 * w] = __builtin_fmaf(bf2f(g & 0xffffu), v[2 * w], bf2f(x & 0xffffu));
                v[2 * w + 1] = __builtin_fmaf(bf2f(g >> 16), v[2 * w + 1], bf2f(x >> 16));
              }
            }
            o[k] = u32x4{pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
          }
          // lanes 16 g16 .. hold columns 32 j + 16 (g16 & 1) + 8 (g16 >> 1) .. + 7
          const int col = n0c + wn * 128 + j * 32 + (g16 & 1) * 16 + (g16 >> 1) * 8;
          put(o[0], o[1], i, col * 2, col < a.N);
        }
        if (i < 2) rows(i + 2);
      }
    } else {
      if (more) {
        origin(tnext);
        prologue();
      }
      // W rows alternate in 16s: quads q = 0, 1 of a fragment are silu's side, q + 2 the factor; 16 output columns each.
      // In place, a row fragment at a time; whether one of its values is far enough for the scaled form is decided once.
      auto glu = [&](int i) __attribute__((always_inline)) {
        float lo = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) lo = fminf(lo, acc[i][j][e]);
        if (__builtin_expect(__any(!(lo >= SILU_FAR)), 0)) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][j][e] = swiglu_f<true>(acc[i][j][e], acc[i][j][8 + e]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][j][e] = swiglu_f<false>(acc[i][j][e], acc[i][j][8 + e]);
        }
      };
      const int ow = n0c / 2 + wn * 64;  // the wave's 64 output columns
      if constexpr (EK == EK_SWIGLU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          glu(i);
#pragma unroll
          for (int jj = 0; jj < 4; jj += 2) {
            u32x4 o[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const f32x16& u = acc[i][jj + k];
              const auto x = __builtin_amdgcn_permlane32_swap(pack2bf(u[0], u[1]), pack2bf(u[4], u[5]), false, false);
              const auto y = __builtin_amdgcn_permlane32_swap(pack2bf(u[2], u[3]), pack2bf(u[6], u[7]), false, false);
              o[k] = u32x4{x[0], y[0], x[1], y[1]};
            }
            const int col = ow + jj * 16 + (g16 & 1) * 16 + (g16 >> 1) * 8;
            put(o[0], o[1], i, col * 2, col < nout);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          glu(i);
          uint32_t mx = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t mj = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) mj = max(mj, abs_bits(acc[i][j][e]));
            mx = max(mx, ow + j * 16 < nout ? mj : 0u);
          }
          const auto s = __builtin_amdgcn_permlane32_swap(mx, mx, false, false);
          if (g2 == 0) xmax[wn * 256 + wm * 128 + i * 32 + r32] = max(s[0], s[1]);
        }
        // raw barrier behind the LDS writes: __syncthreads would wait for the DMA too
        meet();
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ml = wm * 128 + i * 32 + r32;
          const uint32_t b = e8m0_of(max(xmax[ml], xmax[256 + ml]));
          const float r = e8m0_inv(b);
          if (i == 2 * wn + g2) mine = b;  // this wave stores the bytes of row fragments 2 wn and 2 wn + 1
          u32x4 o[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              auto c4 = [&](int j) __attribute__((always_inline)) {
                return pack4_e4m3(acc[i][j][4 * q] * r, acc[i][j][4 * q + 1] * r, acc[i][j][4 * q + 2] * r, acc[i][j][4 * q + 3] * r);
              };
              const auto s = __builtin_amdgcn_permlane32_swap(c4(2 * k), c4(2 * k + 1), false, false);
              o[k][2 * q] = s[0];
              o[k][2 * q + 1] = s[1];
            }
          }
          // o[k]: lanes 0-31 the 16 codes of fragment 2 k, lanes 32-63 of 2 k + 1; behind the exchange lanes 16 g16 ..
          // hold fragment 2 (g16 & 1) + (g16 >> 1)
          const int col = ow + (2 * (g16 & 1) + (g16 >> 1)) * 16;
          put(o[0], o[1], i, col, col < nout);
        }
        const int blk = n0c >> 8;  // the tile's output block
        const __amdgpu_buffer_rsrc_t srs = out_buffer((uint8_t*)a.c_scale + ((int64_t)(blk >> 2) * a.ld_cs + m0c) * 4, (a.M - m0c) * 4);
        const uint32_t so = (uint32_t)((wm * 128 + (2 * wn + g2) * 32 + r32) * 4 + (blk & 3));
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)mine, srs, so, 0, 0);
        if (n0c + BN >= a.N)  // behind the last block the word is 0 (more stores than SN: the waits get stricter)
          for (int z = 1; (blk & 3) + z < 4; ++z) __builtin_amdgcn_raw_buffer_store_b8((uint8_t)0, srs, so + z, 0, 0);
      }
    }
    if (!more) break;
    t = tnext;
    first = false;
  }
}

int cu_count() {
  static int n = 0;  // every GPU of a node is the same
  if (n == 0) {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev);
    n = v > 0 ? v : 256;
  }
  return n;
}

int ek_of(const EchoGemmFp8Args* a) {
  if (a->epilogue == ECHO_EPI_RESID) return a->bias ? EK_RESID_BIAS : EK_RESID;
  if (a->epilogue == ECHO_EPI_SWIGLU) return a->c_scale ? EK_SWIGLU_Q : EK_SWIGLU;
  return a->bias ? EK_BIAS : EK_STORE;
}

// a grid dimension holds fewer than 2^32 threads; a launch of more is cut without an error
bool fits(int64_t workgroups, int threads) { return workgroups * threads <= UINT32_MAX; }

template <int BM, int BN, int WM, int WN, int NS>
int launch_ring(const EchoGemmFp8Args* a, hipStream_t st) {
  const int tm = (a->M + BM - 1) / BM, tn = (a->N + BN - 1) / BN;
  if (!fits((int64_t)tm * tn, 64 * WM * WN)) return ECHO_ESHAPE;
  const dim3 grid(tm * tn), block(64 * WM * WN);
#define ECHO_RING(EK) hipLaunchKernelGGL((gemm_fp8_ring_kernel<BM, BN, WM, WN, NS, EK>), grid, block, 0, st, *a, tm, tn)
  if constexpr (BN == 256) {
    ECHO_RING(EK_SWIGLU_Q);
  } else {
    switch (ek_of(a)) {
      case EK_STORE: ECHO_RING(EK_STORE); break;
      case EK_BIAS: ECHO_RING(EK_BIAS); break;
      case EK_RESID: ECHO_RING(EK_RESID); break;
      case EK_RESID_BIAS: ECHO_RING(EK_RESID_BIAS); break;
      default: ECHO_RING(EK_SWIGLU);
    }
  }
#undef ECHO_RING
  return ECHO_OK;
}

template <int FM, int FN, int KW, int NS>
int launch_few(const EchoGemmFp8Args* a, hipStream_t st) {
  constexpr int BM = FM * 16, BN = FN * 16;
  const int tm = (a->M + BM - 1) / BM, tn = (a->N + BN - 1) / BN;
  if (!fits((int64_t)tm * tn, 64 * KW)) return ECHO_ESHAPE;
  const dim3 grid(tm * tn), block(64 * KW);
#define ECHO_FEW(EK) hipLaunchKernelGGL((gemm_fp8_few_kernel<FM, FN, KW, NS, EK>), grid, block, 0, st, *a, tm, tn)
  switch (ek_of(a)) {
    case EK_STORE: ECHO_FEW(EK_STORE); break;
    case EK_BIAS: ECHO_FEW(EK_BIAS); break;
    case EK_RESID: ECHO_FEW(EK_RESID); break;
    case EK_RESID_BIAS: ECHO_FEW(EK_RESID_BIAS); break;
    default: if constexpr (FN > 1) ECHO_FEW(EK_SWIGLU);
  }
#undef ECHO_FEW
  return ECHO_OK;
}

int launch_ps(const EchoGemmFp8Args* a, hipStream_t st) {
  const int tm = (a->M + 255) / 256, tn = (a->N + 255) / 256;
  const dim3 grid(min(tm * tn, cu_count())), block(256);
#define ECHO_PS(EK) hipLaunchKernelGGL(gemm_fp8_ps_kernel<EK>, grid, block, 0, st, *a, tm, tn, 4)
  switch (ek_of(a)) {
    case EK_STORE: ECHO_PS(EK_STORE); break;
    case EK_BIAS: ECHO_PS(EK_BIAS); break;
    case EK_RESID: ECHO_PS(EK_RESID); break;
    case EK_RESID_BIAS: ECHO_PS(EK_RESID_BIAS); break;
    case EK_SWIGLU: ECHO_PS(EK_SWIGLU); break;
    default: ECHO_PS(EK_SWIGLU_Q);
  }
#undef ECHO_PS
  return ECHO_OK;
}

// The kernels, and what a launch of each costs: rounds of workgroups over the chip (256 CUs) x (1.1 us + K-tiles x the time
// of one). The least is taken. The times of a K-tile are those of one round (K 5888 and 2048, N 2048, M by round); against
// the neighbouring kernels, in us:
//   M    N     K      16x16 16x32 32x32 64x32 64x64 ring64 ring128 ps
//   1    2048  5888    5.5   6.2   7.8  10.0  14.5   23.6   35      50
//   64   2048  2048    6.2   4.4   4.8   5.8   7.9   10.5   15      21
//   157  2048  5888   21.8  16.1  14.3  10.5  15.1   24.1   35      50
//   320  2048  5888   42    27    21    19.2  16.1   24.2   35      51
//   640  2048  2048   46    27    17    14.1  14.3   12.5   16      23
//   157  11776 2048   72    46    28    23.6  23.5   21.5   16.7    26
//   1280 2048  5888  165   101    68    49    50     50     37      61
//   2560 2048  5888  329   200   133    91    79     75     69      62
// quantised SwiGLU:                          ring32  ring64  ps (times of a round of 157 x 2048 x 5888: 37 39 53)
//   320  11776 2048                           33.3    18.8   27.6
//   2560 2048  5888                          111      78     62
enum Kernel { FEW_16x16, FEW_16x32, FEW_32x32, FEW_64x32, FEW_64x64, RING_64, RING_128, RING_32_Q, RING_64_Q, PS };

Kernel pick(const EchoGemmFp8Args* a) {
  struct Row { Kernel k; int bm, bn, ns; };  // ns: a K-tile's time
  static constexpr Row plain[] = {{FEW_16x16, 16, 16, 65}, {FEW_16x32, 16, 32, 80}, {FEW_32x32, 32, 32, 115}, {FEW_64x32, 64, 32, 163},
                                  {FEW_64x64, 64, 64, 270}, {RING_64, 64, 64, 467}, {RING_128, 128, 128, 750}, {PS, 256, 256, 1350}};
  static constexpr Row quant[] = {{RING_32_Q, 32, 256, 780}, {RING_64_Q, 64, 256, 820}, {PS, 256, 256, 1350}};
  const bool glu = a->epilogue == ECHO_EPI_SWIGLU, ps = a->K % BK == 0 && a->K >= 3 * BK && a->K <= PS_KQ * 512;
  const int64_t nkt = (a->K + BK - 1) / BK;
  const int64_t M = (int64_t)a->M * g_policy_num / g_policy_den;  // rows of a one-process run of the whole batch
  Kernel best = PS;
  int64_t least = INT64_MAX;
  auto look = [&](const Row& r) {
    if (r.k == PS ? !ps : r.k == FEW_16x16 && glu) return;  // SwiGLU's W rows come in pairs of 16
    const int64_t tiles = max((M + r.bm - 1) / r.bm, (int64_t)1) * ((a->N + r.bn - 1) / r.bn);
    // two workgroups of RING_64 share a CU, and finish 1.2 times as much
    const int64_t cost = r.k == RING_64 ? max(tiles * 84, (int64_t)25600) * (1100 + nkt * r.ns) / 25600
                                        : (tiles + 255) / 256 * (1100 + nkt * r.ns);
    if (cost < least) { least = cost; best = r.k; }
  };
  if (a->c_scale) for (const Row& r : quant) look(r);
  else for (const Row& r : plain) look(r);
  return best;
}

int check(const EchoGemmFp8Args* a) {
  if (!a) return ECHO_EINVAL;
  if (a->epilogue != ECHO_EPI_STORE && a->epilogue != ECHO_EPI_RESID && a->epilogue != ECHO_EPI_SWIGLU) return ECHO_EINVAL;
  const bool glu = a->epilogue == ECHO_EPI_SWIGLU;
  if (a->c_scale && !glu) return ECHO_EINVAL;
  if (glu && (a->bias || a->aux || a->gate)) return ECHO_EINVAL;
  if (a->epilogue == ECHO_EPI_STORE && (a->aux || a->gate)) return ECHO_EINVAL;
  const int nout = glu ? a->N / 2 : a->N;
  if (a->M < 0 || a->M > INT32_MAX - 255 || a->N <= 0 || a->K <= 0 || a->K % 16 || a->N % (glu ? 32 : 16)) return ECHO_ESHAPE;
  // 32-bit byte offsets inside a tile of up to 256 rows
  if (a->lda < a->K || a->ldw < a->K || a->ldc < nout || a->lda > (1 << 22) || a->ldw > (1 << 22) ||
      a->ldc > (1 << 21)) return ECHO_ESHAPE;
  if (a->ld_as < a->M || a->ld_ws < a->N || (a->c_scale && a->ld_cs < a->M)) return ECHO_ESHAPE;
  if (a->M == 0) return ECHO_OK;
  if ((int64_t)((a->M + 63) / 64) * ((a->N + 63) / 64) > INT32_MAX / 64) return ECHO_ESHAPE;  // workgroups
  if (!a->A || !a->W || !a->C || !a->a_scale || !a->w_scale || (a->epilogue == ECHO_EPI_RESID && !a->aux)) return ECHO_EINVAL;
  if (a->aux && (a->ld_aux < a->N || a->ld_aux > (1 << 21))) return ECHO_ESHAPE;
  if ((uintptr_t)a->A % 16 || (uintptr_t)a->W % 16 || a->lda % 16 || a->ldw % 16 || (uintptr_t)a->C % 16 ||
      a->ldc * (a->c_scale ? 1 : 2) % 16 || (uintptr_t)a->a_scale % 4 || (uintptr_t)a->w_scale % 4 ||
      (uintptr_t)a->c_scale % 4 || (uintptr_t)a->bias % 16 || (uintptr_t)a->gate % 16 || (uintptr_t)a->aux % 16 ||
      (a->aux && a->ld_aux % 8))
    return ECHO_EALIGN;
  return ECHO_OK;
}

}  // namespace

extern "C" {

int32_t echo_gemm_fp8_planned_kernel(const EchoGemmFp8Args* a) {
  const int rc = check(a);
  return rc != ECHO_OK ? rc : a->M == 0 ? PS + 1 : pick(a);
}

int echo_gemm_fp8(const EchoGemmFp8Args* a, void* stream) {
  int rc = check(a);
  if (rc != ECHO_OK || a->M == 0) return rc;
  const hipStream_t st = (hipStream_t)stream;
  switch (pick(a)) {
    case FEW_16x16: rc = launch_few<1, 1, 8, 4>(a, st); break;
    case FEW_16x32: rc = launch_few<1, 2, 8, 3>(a, st); break;
    case FEW_32x32: rc = launch_few<2, 2, 4, 4>(a, st); break;
    case FEW_64x32: rc = launch_few<4, 2, 4, 3>(a, st); break;
    case FEW_64x64: rc = launch_few<4, 4, 4, 2>(a, st); break;
    case RING_64: rc = launch_ring<64, 64, 2, 2, 4>(a, st); break;
    case RING_128: rc = launch_ring<128, 128, 4, 2, 3>(a, st); break;
    case RING_32_Q: rc = launch_ring<32, 256, 1, 4, 3>(a, st); break;
    case RING_64_Q: rc = launch_ring<64, 256, 2, 4, 3>(a, st); break;
    case PS: rc = launch_ps(a, st); break;
  }
  if (rc != ECHO_OK) return rc;
  ECHO_LAUNCH_CHECK();
  return ECHO_OK;
}

}  // extern "C"
