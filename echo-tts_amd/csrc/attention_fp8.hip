// attention_fp8.hip — softmax(q K^T scale) V over up to four segments, each bf16 or an 8-bit cache (fp8.h), * sigmoid(gate).
//
// A cache holds e4m3 codes with one power-of-two scale per (token, head): block = head = 128. An e4m3 value times a
// power of two is exact in bf16, so a tile is converted once, when it goes to LDS (v_cvt_scalef32_pk_bf16_fp8: two
// codes and the scale in one instruction), and everything behind it is the bf16 attention of attention.hip: 4 waves x
// 32 queries of one (row, head), 64-key tiles, scores transposed (S^T = K Q^T, v_mfma_f32_32x32x16_bf16) so that a lane
// holds one query's keys, maximum and sum in fp32, P in bf16 straight from the accumulators into O^T += V^T P.
// What bounds it: 48 rows x 640 queries x 16 heads, half of the ~1350 keys a query own (bf16), half cached: 486-516 us, 750
// TFLOP/s (with bf16 caches attention.hip's kernel takes 437). Under counters (545-595 us, 1.65-1.8 GHz) a SIMD's 983k cycles
// are 360k MFMA and 521k vector (exp2, conversion of codes, sums), of which two waves overlap little. Measured against it, 8
// waves in two groups a phase apart (one in its MFMAs while the other converts and exponentiates, swapped by barriers): 590
// us, though 3 rows of 640 queries take 58 instead of 68 us; fragments read 5 MFMAs ahead: 528 us.
#include "fp8.h"

#include <type_traits>

extern int g_policy_num, g_policy_den;  // echo_set_policy_rows (gemm.hip)
extern int g_attn_split_override;       // echo_attention_set_split (attention.hip)

namespace {

constexpr int KT = 64, QB = 128;
using KArgs = const __attribute__((address_space(4))) EchoAttnFp8Args;

__device__ __forceinline__ int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ float halves_max(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// the lane, opaque: addresses made from it in a loop are made there, and not held (and spilled) from before the loop
__device__ __forceinline__ int opaque_lane() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// Tiles of the segments in order: the state of one walk (scalars; the segment's fields are re-read when it changes)
struct Walk {
  int seg, t0, kend;
  bool causal, coded;
  int ld, sld;                      // bytes from a key to the next
  const uint8_t *k, *v, *ks, *vs;   // at key t0
};

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const uint8_t* uni(const void* p) {
  const uint64_t x = (uint64_t)p;
  return (const uint8_t*)(((uint64_t)(uint32_t)uni((int)(uint32_t)(x >> 32)) << 32) | (uint32_t)uni((int)(uint32_t)x));
}

// loads from a uniform base and a 32-bit byte offset, as global memory: from a plain pointer that was put together from two
// words they are flat ones, which every wait for LDS waits for too
__device__ __forceinline__ uint4 gload16(const uint8_t* p, uint32_t at) {
  const u32x4 x = *(const __attribute__((address_space(1))) u32x4*)((const __attribute__((address_space(1))) uint8_t*)(uintptr_t)p + at);
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint32_t gload1(const uint8_t* p, uint32_t at) {
  return ((const __attribute__((address_space(1))) uint8_t*)(uintptr_t)p)[at];
}

// by value: a ?: between named variables selects their addresses, and they end up in scratch
__device__ __forceinline__ int sel4(int s, int x0, int x1, int x2, int x3) { return s == 0 ? x0 : s == 1 ? x1 : s == 2 ? x2 : x3; }

// keys of each segment that the workgroup's queries may see. Four loads at once (where there is no length, of q): one after
// the other they were half of the time before the first tile
__device__ __forceinline__ void visible(KArgs& a, int row, int q0, int nq, int (&n)[4]) {
  typedef const __attribute__((address_space(1))) int gint;
  int len[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const bool has = s < a.nseg && a.seg[s].len;
    len[s] = *(gint*)(uintptr_t)(has ? (const uint8_t*)(a.seg[s].len + row) : (const uint8_t*)a.q);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int cap = s < a.nseg ? a.seg[s].capacity : 0;
    int x = s < a.nseg && a.seg[s].len ? min(len[s], cap) : cap;
    if (s < a.nseg && a.seg[s].causal) x = min(x, q0 + nq);
    n[s] = uni(max(x, 0));
  }
}

__device__ __forceinline__ void enter(KArgs& a, Walk& w, int row, int head, const int (&n)[4]) {
  do {
    ++w.seg;
    w.kend = sel4(w.seg, n[0], n[1], n[2], n[3]);
  } while (w.kend == 0 && w.seg < 3);
  auto& g = a.seg[w.seg];
  const int b = uni(row % g.batch_mod);
  w.coded = g.k_scale != nullptr;
  const int64_t at = (b * g.ld_batch + head * g.ld_head) * (w.coded ? 1 : 2);
  w.k = uni((const uint8_t*)g.k + at);
  w.v = uni((const uint8_t*)g.v + at);
  w.ld = uni((int)g.ld_tok * (w.coded ? 1 : 2));
  w.causal = g.causal != 0;
  const int64_t sat = b * g.s_batch + head * g.s_head;
  w.ks = uni((const uint8_t*)g.k_scale + sat);
  w.vs = uni((const uint8_t*)g.v_scale + sat);
  w.sld = w.coded ? uni((int)g.s_tok) : 0;
  w.t0 = 0;
}
__device__ __forceinline__ void step(KArgs& a, Walk& w, int row, int head, const int (&n)[4]) {
  w.t0 += KT;
  if (w.t0 >= w.kend) {
    enter(a, w, row, head, n);
  } else {
    w.k += KT * w.ld;
    w.v += KT * w.ld;
    w.ks += KT * w.sld;
    w.vs += KT * w.sld;
  }
}

// 16 codes and their scale -> 16 bf16
__device__ __forceinline__ void decode16(const uint4& c, uint32_t byte, uint4& lo, uint4& hi) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf2;
  const float s = __uint_as_float(byte << 23);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = __builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], s, false));
    r[2 * i + 1] = __builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], s, true));
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// 4 columns of one query: v / l, times sigmoid of the gate's u, one rounding; l == 0 (nothing visible): zeros; NaN stays
template <class Args>
__device__ __forceinline__ uint2 finish4(const Args& a, float4 v, float l, uint2 u) {
  const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
  v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  if (a.gate) {
    v.x *= sigmoid_f(bf2f(u.x & 0xffffu));
    v.y *= sigmoid_f(bf2f(u.x >> 16));
    v.z *= sigmoid_f(bf2f(u.y & 0xffffu));
    v.w *= sigmoid_f(bf2f(u.y >> 16));
  }
  return make_uint2(pack2bf(v.x, v.y), pack2bf(v.z, v.w));
}
template <class Args>
__device__ __forceinline__ void write_out4(const Args& a, const float (&v)[4], float l, int row, int qrow, int head, int qi, int c) {
  uint2 u = make_uint2(0, 0);
  if (a.gate) u = *(const uint2*)((const bf16_t*)a.gate + qrow * a.g_ld_batch + (int64_t)qi * a.g_ld_tok + head * 128 + c * 4);
  *(uint2*)((bf16_t*)a.out + row * a.o_ld_batch + (int64_t)qi * a.o_ld_tok + head * 128 + c * 4) =
      finish4(a, make_float4(v[0], v[1], v[2], v[3]), l, u);
}

// SPLIT: workgroup (q block, split, row, head) walks its share of the tiles and stores O (fp32, unnormalised), the
// reference of its exponents (exp2 units) and the sum; attn_fp8_join_kernel joins the parts.
//
// The exponents' reference is the maximum of the first tile, and stays: a later score above it only makes P larger than 1,
// and fp32 sums and a bf16 P hold any power of two up to 2^127 with the same relative precision. So the loop has no
// maximum, no rescaling and no branch around O (which the compiler turns into 64 moves a tile). If a query's sum passes
// 2^60 (a score 2^60 above the first tile's, or not finite), one of its sums in O 2^100 (large values at such a score; up to
// 64 parts of it still add up in the join) or its first tile has only -inf, the workgroup walks its tiles once more with the
// running maximum (SAFE); so it does at once where a segment is causal, whose first tile may show a query nothing.
template <bool SPLIT>
__global__ void __launch_bounds__(256, 2) attn_fp8_kernel(EchoAttnFp8Args arg, float* ws, int nsplit) {
  (void)arg;
  KArgs& a = *(KArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  __shared__ __attribute__((aligned(16))) bf16_t lds[2 * 2 * KT * 128];  // [buffer][K | V][64 keys][128]
  __shared__ int again[4];
  __shared__ float sums[4][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, ql = lane & 31;
  const int nqb = (a.n_q + QB - 1) / QB;
  // an XCD's workgroups are consecutive ones: the q blocks of a (row, head), then the rows that share its caches
  const int nwg = gridDim.x, q8 = nwg >> 3, r8 = nwg & 7, xcd = blockIdx.x & 7;
  int L = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
  const int qb = uni(L % nqb);
  L /= nqb;
  const int sp = SPLIT ? uni(L % nsplit) : 0;
  if (SPLIT) L /= nsplit;
  const int row = uni(L % a.rows), head = uni(L / a.rows);
  const int q0 = qb * QB, qw = q0 + w * 32, qi = qw + ql;
  const int qrow = uni(a.q_batch_mod > 0 ? row % a.q_batch_mod : row);

  bf16x8 qf[8];
  {
    const bf16_t* qp = (const bf16_t*)a.q + qrow * a.q_ld_batch + (int64_t)min(qi, a.n_q - 1) * a.q_ld_tok + head * 128;
#pragma unroll
    for (int ds = 0; ds < 8; ++ds) qf[ds] = *(const bf16x8*)(qp + 16 * ds + 8 * h2);
  }
  int nv[4];
  visible(a, row, q0, QB, nv);
  const int ntiles = (nv[0] + KT - 1) / KT + (nv[1] + KT - 1) / KT + (nv[2] + KT - 1) / KT + (nv[3] + KT - 1) / KT;
  const int tb = SPLIT ? uni((int)((int64_t)sp * ntiles / nsplit)) : 0;
  const int te = SPLIT ? uni((int)((int64_t)(sp + 1) * ntiles / nsplit)) : ntiles;
  int any_causal = 0;
  for (int s = 0; s < a.nseg; ++s) any_causal |= a.seg[s].causal;

  f32x16 o[4];
  float m_run, l_run;
  const float sl2 = a.scale * 1.4426950408889634f;
  Walk ld;

  // LDS byte addresses of the buffer in turn ([K 16 KB | V 16 KB], two of them: they alternate by bit 15): K fragment
  // reads (row ql, chunk 2 ds + h2; 32 rows on: + 8192), transposed V reads (rows r0 = 4 h2 + q4 and r0 + 8, chunk by d;
  // 16 rows on: + 4096), and where this thread puts its codes (row tid / 8, and 32 on). All swizzled by chunk ^ swz(row).
  typedef __attribute__((address_space(3))) uint8_t lds8;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr_of(lds));
  uint32_t ka, va[2], pa, pb, buf = 0;
  {
    ka = lds0 + (uint32_t)(ql * 256 + ((h2 ^ swz(ql)) * 16));
    const int g = lane >> 4, q4 = (lane & 15) >> 2, p4 = lane & 3, r0 = 4 * h2 + q4;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      va[h] = lds0 + 16384 + (uint32_t)((r0 + 8 * h) * 256 + (((2 * (g & 1) + (p4 >> 1)) ^ swz(r0 + 8 * h)) * 16) + (p4 & 1) * 8);
    const int r = tid >> 3, c = 2 * (tid & 7);
    pa = lds0 + (uint32_t)(r * 256 + ((c ^ swz(r)) * 16));
    pb = lds0 + (uint32_t)(r * 256 + (((c + 1) ^ swz(r)) * 16));
  }
  auto flip = [&]() __attribute__((always_inline)) {
    buf ^= 32768;
    ka ^= 32768;
    va[0] ^= 32768;
    va[1] ^= 32768;
    pa ^= 32768;
    pb ^= 32768;
  };
  auto put16 = [&](uint32_t at, const uint4& x) __attribute__((always_inline)) { *(__attribute__((address_space(3))) u32x4*)(lds8*)(uintptr_t)at = u32x4{x.x, x.y, x.z, x.w}; };

  // The tiles from ti on as long as they are of one type. C: codes go through registers (16-B pieces, 8 a row, and their
  // scale bytes), requested a tile ahead, and are converted when they are put into LDS; bf16 goes there by LDS-DMA, the
  // swizzle applied to the source. Rows past the visible keys repeat the last one.
  auto run = [&](int ti, auto coded, auto safe) __attribute__((always_inline)) -> int {
    constexpr bool C = decltype(coded)::value, SAFE = decltype(safe)::value;
    uint4 kr[2], vr[2];
    uint32_t sb;
    int nlim, nt0;  // of the tile on its way: visible keys from its first, and its place in the segment
    bool ncausal;
    auto load = [&](uint32_t to) __attribute__((always_inline)) {
      const int lane = opaque_lane(), tid = w * 64 + lane;  // or every piece's place is held (and spilled)
      ncausal = ld.causal;
      nt0 = ld.t0;
      nlim = ld.kend - ld.t0;
      const int last = nlim - 1;
      const uint32_t sd = (uint32_t)ld.ld;
      const uint8_t *kp = uni(ld.k), *vp = uni(ld.v);
      if constexpr (C) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t at = __umul24((uint32_t)min((tid >> 3) + i * 32, last), sd) + (tid & 7) * 16;
          kr[i] = gload16(kp, at);
          vr[i] = gload16(vp, at);
        }
        // the wave's 32 scale bytes in one load (keys' rows 8 w .. and 32 on, then values'), handed out when they are put
        sb = gload1(lane & 16 ? uni(ld.vs) : uni(ld.ks), __umul24((uint32_t)min(w * 8 + (lane & 7) + (lane & 8) * 4, last), (uint32_t)ld.sld));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (i * 4 + w) * 4 + (lane >> 4);
          const uint32_t off = __umul24((uint32_t)min(r, last), sd) + ((lane & 15) ^ swz(r)) * 16;
          const uint32_t dst = lds0 + to + (uint32_t)((i * 4 + w) * 1024);
          glds16s(kp, off, dst);
          glds16s(vp, off, dst + 16384);
        }
      }
    };
    load(buf);
    bool more = true;
#pragma unroll 1
    while (more) {
      if constexpr (C) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 lo, hi;
          decode16(kr[i], (uint32_t)__builtin_amdgcn_ds_bpermute((lane >> 3) * 4 + i * 32, (int)sb), lo, hi);
          put16(pa + i * 8192, lo);
          put16(pb + i * 8192, hi);
          decode16(vr[i], (uint32_t)__builtin_amdgcn_ds_bpermute((lane >> 3) * 4 + 64 + i * 32, (int)sb), lo, hi);
          put16(pa + 16384 + i * 8192, lo);
          put16(pb + 16384 + i * 8192, hi);
        }
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __syncthreads();  // tile ti is in LDS, and every wave is done reading tile ti - 1: its buffer takes tile ti + 1
      const int lim0 = nlim, t0 = nt0;
      const bool causal = ncausal, head_tile = ti == tb;
      ++ti;
      more = ti < te;
      if (more) {
        step(a, ld, row, head, nv);
        more = ld.coded == C;
        if (more) load(buf ^ 32768);
      }
      f32x16 st[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[kk][r] = 0.f;
#pragma unroll
        for (int ds = 0; ds < 8; ++ds) {
          const bf16x8 kf = *(__attribute__((address_space(3))) const bf16x8*)(lds8*)(uintptr_t)((ka ^ (ds * 32)) + kk * 8192);
          st[kk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ds], st[kk], 0, 0, 0);
        }
      }
      // K fragments are read 4 MFMAs ahead
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 2);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 2);
        if (i + 4 < 16) __builtin_amdgcn_sched_group_barrier(0x100, 1, 2);
      }
      // lane: query ql, keys t0 + kk * 32 + (r & 3) + 8 (r >> 2) + 4 h2
      if ((SAFE && causal) || lim0 < KT) {
        const int lim = (SAFE && causal ? min(lim0, qi + 1 - t0) : lim0) - 4 * h2;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = kk * 32 + (r & 3) + 8 * (r >> 2);
            st[kk][r] = key < lim ? st[kk][r] : -INFINITY;
          }
      }
      if (SAFE || head_tile) {
        float mx = -INFINITY;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int r = 0; r < 16; r += 2)
            mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, st[kk][r]), st[kk][r + 1]);
        mx = halves_max(mx);
        if constexpr (SAFE) {
          const float mn = __builtin_elementwise_maximum(m_run, mx);
          const float al = __builtin_amdgcn_exp2f(__builtin_fmaf(m_run, sl2, mn == -INFINITY ? 0.f : -mn * sl2));
          l_run *= al;
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= al;
          m_run = mn;
        } else {
          m_run = mx;
        }
      }
      const float msc = m_run == -INFINITY ? 0.f : -m_run * sl2;
      float ps[2] = {0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[kk][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kk][r], sl2, msc));
#pragma unroll
        for (int r = 0; r < 16; ++r) ps[kk] += st[kk][r];
      }
      l_run += ps[0] + ps[1];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          bf16x8 pf;
#pragma unroll
          for (int j = 0; j < 8; ++j) pf[j] = (__bf16)st[kk][8 * s2 + j];
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            typedef __attribute__((ext_vector_type(8))) short s16x8;
            typedef __attribute__((address_space(3))) s16x4 lds64;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64*)(lds8*)(uintptr_t)((va[0] ^ (d * 64)) + kk * 8192 + s2 * 4096));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64*)(lds8*)(uintptr_t)((va[1] ^ (d * 64)) + kk * 8192 + s2 * 4096));
            const s16x8 v8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v8), pf, o[d], 0, 0, 0);
          }
        }
      // V^T fragments (two transposed reads each) 2 MFMAs ahead
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 3);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 3);
        if (i + 2 < 16) __builtin_amdgcn_sched_group_barrier(0x100, 2, 3);
      }
      flip();
    }
    return ti;
  };
  auto walk = [&](auto safe) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    m_run = -INFINITY;
    l_run = 0.f;
    ld = Walk{-1, 0, 0, false, false, 0, 0, nullptr, nullptr, nullptr, nullptr};
    if (tb >= te) return;
    enter(a, ld, row, head, nv);
    for (int i = 0; i < tb; ++i) step(a, ld, row, head, nv);
    int ti = tb;
    while (ti < te) ti = ld.coded ? run(ti, std::true_type{}, safe) : run(ti, std::false_type{}, safe);
  };
  bool redo = any_causal != 0;
  if (!redo) {
    walk(std::false_type{});
    float most = 0.f;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = __builtin_elementwise_maximum(most, __builtin_fabsf(o[d][r]));
    if (lane == 0) again[w] = 0;
    if (__any(!(l_run <= 0x1p60f) || m_run == -INFINITY || !(most <= 0x1p100f)) && lane == 0) again[w] = 1;
    __syncthreads();
    redo = uni(again[0] | again[1] | again[2] | again[3]) != 0;
    __syncthreads();
  }
  if (redo) walk(std::true_type{});

  // lane: query qi, columns 32 d + 8 rg + 4 h2 .. + 3 in o[d][4 rg ..]
  const float l = halves_sum(l_run);
  if constexpr (SPLIT) {
    if (qi >= a.n_q) return;
    // parts [split][row][head]: O as [32 column quads][query][4], then (m, l) of every query
    const int64_t it = ((int64_t)sp * a.rows + row) * a.heads + head;
    float* wo = ws + it * 128 * a.n_q;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg)
        *(float4*)(wo + ((int64_t)(d * 8 + 2 * rg + h2) * a.n_q + qi) * 4) =
            make_float4(o[d][4 * rg], o[d][4 * rg + 1], o[d][4 * rg + 2], o[d][4 * rg + 3]);
    if (h2 == 0)
      *(float2*)(ws + (int64_t)nsplit * a.rows * a.heads * 128 * a.n_q + (it * a.n_q + qi) * 2) =
          make_float2(m_run == -INFINITY ? -INFINITY : m_run * sl2, l);
  } else {
    // through LDS ([query][column quad ^ query]; the wave's own part, every wave is done with the tiles), so that gate and
    // output go in whole rows: 16 lanes x 16 B a query
    uint4 gt[8] = {};
    const int ql4 = lane >> 4, c = 2 * (lane & 15);
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        gt[i] = *(const uint4*)((const bf16_t*)a.gate + qrow * a.g_ld_batch + (int64_t)min(qw + i * 4 + ql4, a.n_q - 1) * a.g_ld_tok + head * 128 + c * 4);
    }
    __syncthreads();
    float4* const part = (float4*)lds + w * 1024;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg)
        part[ql * 32 + ((d * 8 + 2 * rg + h2) ^ ql)] = make_float4(o[d][4 * rg], o[d][4 * rg + 1], o[d][4 * rg + 2], o[d][4 * rg + 3]);
    sums[w][ql] = l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int q = i * 4 + ql4;
      const uint2 y0 = finish4(a, part[q * 32 + (c ^ q)], sums[w][q], make_uint2(gt[i].x, gt[i].y));
      const uint2 y1 = finish4(a, part[q * 32 + ((c + 1) ^ q)], sums[w][q], make_uint2(gt[i].z, gt[i].w));
      if (qw + q < a.n_q)
        *(uint4*)((bf16_t*)a.out + row * a.o_ld_batch + (int64_t)(qw + q) * a.o_ld_tok + head * 128 + c * 4) = make_uint4(y0.x, y0.y, y1.x, y1.y);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few queries
// A workgroup of 8 waves has 32 queries of one (row, head); the waves share out the 32-key tiles (w, w + 8, ..) and walk
// them on their own, without a barrier, each with a running maximum, sum and O; at the end the 8 parts are joined through
// LDS. With few queries the caches are read once and little else happens, so what counts is bytes in flight: K and V of a
// wave's next tile (8 KB of codes) are requested as soon as this tile's are consumed, 64 KB a CU.
// Both go through the wave's own 16 KB of LDS, requested in whole rows (8 lanes a row of codes): straight from memory, a
// fragment's neighbouring lanes are different rows, which takes L1 four times the cycles and was the bound (1 row of 2048
// keys: 20 us). Keys stay codes there: the product over d does not care for its order, so lane (key, half) takes bytes
// 32 i + 16 half .. + 15 of its row, and q is permuted alike. MFMA time matters little here: P is kept as two bf16 (value
// and remainder, 16 bits), so that the only rounding worth naming is the output's.
// 16 rows x 16 heads x 1 query: 2048 keys 28 us (4.8 TB/s), 4096 keys 49 us (5.5 TB/s); a tile's chain takes a wave 2 us,
// which is the bound where a wave has few tiles (1 row, 512 keys 8.3 us).
constexpr int FW = 8, FK = 32;  // waves, keys a tile

struct Seg {  // one wave's current segment (scalars)
  int seg, kend;
  bool causal, coded;
  int ld, sld;
  const uint8_t *k, *v, *ks, *vs;
};

template <bool SPLIT>
__global__ void __launch_bounds__(64 * FW, 2) attn_fp8_few_kernel(EchoAttnFp8Args arg, float* ws, int nsplit) {
  (void)arg;
  KArgs& a = *(KArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  __shared__ __attribute__((aligned(16))) uint8_t lds[FW * 16384];  // a wave's V and K tiles (8 KB each); its part of O at the end
  __shared__ float2 ml[FW][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uni(tid >> 6);
  const int h2 = lane >> 5, ql = lane & 31;
  const int nqb = (a.n_q + 31) / 32;
  int L = blockIdx.x;
  const int qb = L % nqb;
  L /= nqb;
  const int sp = SPLIT ? L % nsplit : 0;
  if (SPLIT) L /= nsplit;
  const int row = uni(L % a.rows), head = uni(L / a.rows);
  const int q0 = qb * 32, qi = q0 + ql, nq = min(a.n_q - q0, 32);
  const int qrow = a.q_batch_mod > 0 ? row % a.q_batch_mod : row;

  bf16x8 qf[8];
  {
    const bf16_t* qp = (const bf16_t*)a.q + qrow * a.q_ld_batch + (int64_t)min(qi, a.n_q - 1) * a.q_ld_tok + head * 128;
#pragma unroll
    for (int ds = 0; ds < 8; ++ds) qf[ds] = *(const bf16x8*)(qp + (ds >> 1) * 32 + h2 * 16 + (ds & 1) * 8);
  }
  int nv[4];
  visible(a, row, q0, 32, nv);
  const int n0 = nv[0], n1 = nv[1], n2 = nv[2], n3 = nv[3];
  const int c0 = (n0 + FK - 1) / FK, c1 = c0 + (n1 + FK - 1) / FK, c2 = c1 + (n2 + FK - 1) / FK, c3 = c2 + (n3 + FK - 1) / FK;
  const int tb = SPLIT ? (int)((int64_t)sp * c3 / nsplit) : 0, te = SPLIT ? (int)((int64_t)(sp + 1) * c3 / nsplit) : c3;

  Seg g{-1, 0, false, false, 0, 0, nullptr, nullptr, nullptr, nullptr};
  int t0 = 0;
  auto locate = [&](int idx) __attribute__((always_inline)) {  // tile idx of the flat list
    const int sg = uni(idx < c0 ? 0 : idx < c1 ? 1 : idx < c2 ? 2 : 3);
    t0 = uni((idx - sel4(sg, 0, c0, c1, c2)) * FK);
    if (sg == g.seg) return;
    g.seg = sg;
    g.kend = sel4(sg, n0, n1, n2, n3);
    auto& x = a.seg[sg];
    const int b = row % x.batch_mod;
    g.coded = uni(x.k_scale != nullptr) != 0;
    g.causal = uni(x.causal) != 0;
    const int64_t at = (b * x.ld_batch + head * x.ld_head) * (g.coded ? 1 : 2), sat = b * x.s_batch + head * x.s_head;
    g.k = uni((const uint8_t*)x.k + at);
    g.v = uni((const uint8_t*)x.v + at);
    g.ks = uni((const uint8_t*)x.k_scale + sat);
    g.vs = uni((const uint8_t*)x.v_scale + sat);
    g.ld = uni((int)x.ld_tok * (g.coded ? 1 : 2));
    g.sld = uni((int)x.s_tok);
  };

  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float sl2 = a.scale * 1.4426950408889634f;
  bf16_t* const Vs = (bf16_t*)(lds + w * 16384);
  uint8_t* const Ks = lds + w * 16384 + 8192;

  int idx = tb + w;
  // the wave's tiles from idx on as long as they are of one type (C: codes)
  auto run = [&](auto coded) __attribute__((always_inline)) {
    constexpr bool C = decltype(coded)::value;
    // codes are requested a tile ahead; bf16 (a row's own few keys, as a rule) as it is needed
    uint4 kr[4], vr[4];
    uint32_t kb = 0, vb[4] = {};
    auto load = [&]() __attribute__((always_inline)) {
      if constexpr (C) {
        const int lane = opaque_lane();
        const int last = g.kend - 1 - t0;
        const uint8_t *kp = uni(g.k + (int64_t)t0 * g.ld), *vp = uni(g.v + (int64_t)t0 * g.ld);
        const uint8_t *ksp = uni(g.ks + (int64_t)t0 * g.sld), *vsp = uni(g.vs + (int64_t)t0 * g.sld);
        const uint32_t ld = (uint32_t)g.ld;
        kb = gload1(ksp, (uint32_t)min(lane & 31, last) * (uint32_t)g.sld);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t r = (uint32_t)min(i * 8 + (lane >> 3), last), at = r * ld + (lane & 7) * 16;
          kr[i] = gload16(kp, at);
          vr[i] = gload16(vp, at);
          vb[i] = gload1(vsp, r * (uint32_t)g.sld);
        }
      }
    };
    load();
    for (bool more = true; more; idx += FW) {
      const int lim = g.kend - t0, tt = t0;  // this tile's
      const int lane = opaque_lane(), ql = lane & 31, h2 = lane >> 5, q4 = (lane & 15) >> 2, p4 = lane & 3;
      const bool causal = g.causal;
      f32x16 st;
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = 0.f;
      if constexpr (C) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 lo, hi;
          const int r = i * 8 + (lane >> 3), p = 2 * (lane & 7);
          *(uint4*)(Ks + r * 128 + ((lane & 7) ^ (r & 7)) * 16) = kr[i];
          decode16(vr[i], vb[i], lo, hi);
          *(uint4*)(Vs + r * 128 + ((p ^ swz(r)) * 8)) = lo;
          *(uint4*)(Vs + r * 128 + (((p + 1) ^ swz(r)) * 8)) = hi;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 lo, hi;
          decode16(*(const uint4*)(Ks + ql * 128 + ((2 * i + h2) ^ (ql & 7)) * 16), kb, lo, hi);
          st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, lo), qf[2 * i], st, 0, 0, 0);
          st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, hi), qf[2 * i + 1], st, 0, 0, 0);
        }
      } else {
        const uint8_t *kp = uni(g.k + (int64_t)t0 * g.ld), *vp = uni(g.v + (int64_t)t0 * g.ld);
        const uint32_t ld = (uint32_t)g.ld;
        uint4 x[8];
        auto fill = [&](const uint8_t* from, uint8_t* to) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = gload16(from, (uint32_t)min(i * 4 + (lane >> 4), lim - 1) * ld + (lane & 15) * 16);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 4);
            *(uint4*)(to + r * 256 + ((lane & 15) ^ swz(r)) * 16) = x[i];
          }
        };
        fill(kp, Ks);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              *(const bf16x8*)(Ks + ql * 256 + (((i >> 1) * 4 + h2 * 2 + (i & 1)) ^ swz(ql)) * 16), qf[i], st, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        fill(vp, (uint8_t*)Vs);
      }
      __builtin_amdgcn_sched_barrier(0);
      more = idx + FW < te;
      if (more) {
        locate(idx + FW);
        more = g.coded == C;
        if (more) load();
      }
      __builtin_amdgcn_sched_barrier(0);
      // lane: query ql, keys tt + (r & 3) + 8 (r >> 2) + 4 h2
      if (causal || lim < FK) {
        const int lm = (causal ? min(lim, qi + 1 - tt) : lim) - 4 * h2;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = (r & 3) + 8 * (r >> 2) < lm ? st[r] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; r += 2) mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, st[r]), st[r + 1]);
      mx = halves_max(mx);
      if (__any(m_run == -INFINITY || (mx - m_run) * sl2 > 8.0f)) {
        const float mn = fmaxf(m_run, mx);
        const float al = __builtin_amdgcn_exp2f(__builtin_fmaf(m_run, sl2, mn == -INFINITY ? 0.f : -mn * sl2));
        l_run *= al;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= al;
        m_run = mn;
      }
      const float msc = m_run == -INFINITY ? 0.f : -m_run * sl2;
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], sl2, msc));
        ps += st[r];
      }
      l_run += ps;
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        bf16x8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ph[j] = (__bf16)st[8 * s2 + j];
          pl[j] = (__bf16)(st[8 * s2 + j] - (float)ph[j]);
        }
        const int r0 = 16 * s2 + 4 * h2 + q4, r1 = r0 + 8;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int ch = 4 * d + 2 * ((lane >> 4) & 1) + (p4 >> 1);
          typedef __attribute__((ext_vector_type(8))) short s16x8;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(Vs + r0 * 128 + ((ch ^ swz(r0)) * 8) + (p4 & 1) * 4));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(Vs + r1 * 128 + ((ch ^ swz(r1)) * 8) + (p4 & 1) * 4));
          const bf16x8 v8 = __builtin_bit_cast(bf16x8, (s16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v8, ph, o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v8, pl, o[d], 0, 0, 0);
        }
      }
    }
  };
  while (idx < te) {
    locate(idx);
    if (g.coded) run(std::true_type{}); else run(std::false_type{});
  }

  // join: part w as [query][column quad ^ query], (m in exp2 units, l)
  const float l = halves_sum(l_run);
  float4* const part = (float4*)(lds + w * 16384);
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg)
      part[ql * 32 + ((d * 8 + 2 * rg + h2) ^ ql)] = make_float4(o[d][4 * rg], o[d][4 * rg + 1], o[d][4 * rg + 2], o[d][4 * rg + 3]);
  if (h2 == 0) ml[w][ql] = make_float2(m_run == -INFINITY ? -INFINITY : m_run * sl2, l);
  __syncthreads();
  for (int u = tid; u < nq * 32; u += 64 * FW) {
    const int q = u >> 5, c = u & 31;
    float m = -INFINITY;
#pragma unroll
    for (int p = 0; p < FW; ++p) m = __builtin_elementwise_maximum(m, ml[p][q].x);
    float v[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
    for (int p = 0; p < FW; ++p) {
      const float2 x = ml[p][q];
      const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
      const float4 y = ((const float4*)(lds + p * 16384))[q * 32 + (c ^ q)];
      ls = __builtin_fmaf(x.y, f, ls);
      v[0] = __builtin_fmaf(y.x, f, v[0]);
      v[1] = __builtin_fmaf(y.y, f, v[1]);
      v[2] = __builtin_fmaf(y.z, f, v[2]);
      v[3] = __builtin_fmaf(y.w, f, v[3]);
    }
    if constexpr (SPLIT) {
      const int64_t it = ((int64_t)sp * a.rows + row) * a.heads + head;
      *(float4*)(ws + (it * 32 + c) * a.n_q * 4 + (int64_t)(q0 + q) * 4) = make_float4(v[0], v[1], v[2], v[3]);
      if (c == 0)
        *(float2*)(ws + (int64_t)nsplit * a.rows * a.heads * 128 * a.n_q + (it * a.n_q + q0 + q) * 2) = make_float2(m, ls);
    } else {
      write_out4(a, v, ls, row, qrow, head, q0 + q, c);
    }
  }
}

// out = sum_s O_s 2^(m_s - m) / sum_s l_s 2^(m_s - m), gated: one thread per (row, head, column quad, query)
__global__ void __launch_bounds__(256) attn_fp8_join_kernel(EchoAttnFp8Args a, const float* __restrict__ ws, int nsplit) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = (int64_t)32 * a.n_q;
  if (x >= per * a.rows * a.heads) return;
  const int rh = (int)(x / per), rest = (int)(x - rh * per), c = rest / a.n_q, qi = rest - c * a.n_q;
  const int row = rh / a.heads, head = rh - row * a.heads;
  const int64_t parts = (int64_t)a.rows * a.heads;
  const float* ml = ws + nsplit * parts * 128 * a.n_q;
  const float* const o = ws + ((int64_t)rh * 32 + c) * a.n_q * 4 + (int64_t)qi * 4;
  float m = -INFINITY, v[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int s0 = 0; s0 < nsplit; s0 += 8) {  // 8 parts' loads in flight
    float2 p[8];
    float4 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = min(s0 + k, nsplit - 1);
      p[k] = *(const float2*)(ml + ((s * parts + rh) * a.n_q + qi) * 2);
      u[k] = *(const float4*)(o + s * parts * 128 * a.n_q);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) mn = fmaxf(mn, p[k].x);
    const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= al;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= al;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = s0 + k >= nsplit || p[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p[k].x - m);
      l = __builtin_fmaf(p[k].y, f, l);
      v[0] = __builtin_fmaf(u[k].x, f, v[0]);
      v[1] = __builtin_fmaf(u[k].y, f, v[1]);
      v[2] = __builtin_fmaf(u[k].z, f, v[2]);
      v[3] = __builtin_fmaf(u[k].w, f, v[3]);
    }
  }
  write_out4(a, v, l, row, a.q_batch_mod > 0 ? row % a.q_batch_mod : row, head, qi, c);
}

int64_t keys_of(const EchoAttnFp8Args* a) {
  int64_t n = 0;
  for (int s = 0; s < a->nseg; ++s) n += a->seg[s].capacity;
  return n;
}

// workgroups of the launch as a one-process run of the whole batch would have them (echo_set_policy_rows)
int64_t policy(int64_t items) { return items * g_policy_num / g_policy_den; }

// Queries a workgroup: 32 (few) or 128. Where the keys are not many and 32 queries a workgroup make no more than a round of
// workgroups, more queries go to the kernel for few as well. us, 16 heads, few | many:
//   rows x queries x keys   1x64x1024 12.1 | 11.8   1x192x512 10.2 | 13.8   4x64x1024 15.2 | 19.0   4x128x1024 19.9 | 24.6
//   more keys               4x64x2368 27.0 | 23.3   4x96x6000 59 | 42     more workgroups   16x33x512 23.5 | 15.0
bool few(const EchoAttnFp8Args* a) {
  return a->n_q <= 32 || (keys_of(a) <= 2048 && policy(((a->n_q + 31) / 32) * (int64_t)a->heads * a->rows) <= 256);
}
int64_t items_of(const EchoAttnFp8Args* a) {
  const int qb = few(a) ? 32 : QB;
  return (int64_t)((a->n_q + qb - 1) / qb) * a->heads * a->rows;
}

// a grid dimension holds fewer than 2^32 threads; a launch of more is cut without an error
bool fits(const EchoAttnFp8Args* a, int64_t nsplit) {
  return items_of(a) <= UINT32_MAX / ((few(a) ? 64 * FW : 256) * max(nsplit, (int64_t)1)) &&
         (nsplit <= 1 || (int64_t)a->rows * a->heads * 32 * a->n_q <= UINT32_MAX - 255);
}

bool bad16(const void* p, int64_t bytes) { return (uintptr_t)p % 16 || bytes % 16; }

int check(const EchoAttnFp8Args* a) {
  if (!a) return ECHO_EINVAL;
  if (a->rows < 0 || a->n_q < 0 || a->heads <= 0 || a->nseg < 0 || a->nseg > 4 || a->q_batch_mod < 0) return ECHO_ESHAPE;
  if (a->rows == 0 || a->n_q == 0) return ECHO_OK;
  if (a->n_q > INT32_MAX - QB || (int64_t)a->rows * a->heads > INT32_MAX) return ECHO_ESHAPE;
  if (!a->q || !a->out || !(a->scale > 0.f)) return ECHO_EINVAL;
  if (bad16(a->q, a->q_ld_tok * 2) || a->q_ld_batch % 8 || bad16(a->out, a->o_ld_tok * 2) || a->o_ld_batch % 8 ||
      (a->gate && (bad16(a->gate, a->g_ld_tok * 2) || a->g_ld_batch % 8)))
    return ECHO_EALIGN;
  int64_t keys = 0;
  for (int s = 0; s < a->nseg; ++s) {
    const EchoKVSegmentFp8& g = a->seg[s];
    if (g.capacity < 0) return ECHO_ESHAPE;
    if (g.capacity == 0) continue;
    if (!g.k || !g.v || (g.k_scale == nullptr) != (g.v_scale == nullptr)) return ECHO_EINVAL;
    if (g.batch_mod <= 0) return ECHO_ESHAPE;
    const int es = g.k_scale ? 1 : 2;
    if (bad16(g.k, g.ld_tok * es) || bad16(g.v, g.ld_batch * es) || g.ld_head * es % 16) return ECHO_EALIGN;
    // rows inside a tile are found by 24-bit products of bytes
    if (g.ld_tok < 0 || g.ld_tok >= (1 << 24) / es || (es == 1 && (g.s_tok < 0 || g.s_tok >= (1 << 24)))) return ECHO_ESHAPE;
    keys += g.capacity;
  }
  if (keys > INT32_MAX - 256 || !fits(a, 1)) return ECHO_ESHAPE;
  return ECHO_OK;
}

}  // namespace

extern "C" {

int32_t echo_attention_fp8_pick_split(const EchoAttnFp8Args* a) {
  if (check(a) != ECHO_OK || a->rows == 0 || a->n_q == 0) return 1;
  if (g_attn_split_override >= 0) return max(1, min(g_attn_split_override, 16));
  const int64_t items = max(policy(items_of(a)), (int64_t)1), tiles = (keys_of(a) + KT - 1) / KT;
  // The parts cost a pass of their own: split from 1024 keys on (few queries; 1536 for many), if it fills the chip. us, 16
  // heads, unsplit | split: 1 query of 1 row 1024 keys 12.6 | 9.3, 2048 21.4 | 9.8; 640 queries of 1 row 512 keys 14.8 | 24.3
  if (items >= 192) return 1;
  int64_t n;
  if (few(a)) {
    n = tiles < 16 ? 1 : 256 / items;
    if (n > tiles / 4) n = tiles / 4;
    if (n == 2 && tiles < 32) n = 1;  // 64 queries of 4 rows, 1024 keys: 15.3 | 18.4
  } else {
    n = tiles < 24 ? 1 : 512 / items;
    if (n > tiles / 2) n = tiles / 2;
  }
  if (n > 16) n = 16;
  return n < 1 ? 1 : (int32_t)n;
}

int64_t echo_attention_fp8_ws_bytes(const EchoAttnFp8Args* a, int32_t nsplit) {
  if (nsplit <= 1 || check(a) != ECHO_OK) return 0;
  return (int64_t)nsplit * a->rows * a->heads * a->n_q * (128 + 2) * 4;
}

int echo_attention_fp8(const EchoAttnFp8Args* a, int32_t nsplit, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = check(a);
  if (rc != ECHO_OK || a->rows == 0 || a->n_q == 0) return rc;
  if (nsplit > 64) return ECHO_EINVAL;
  if (!fits(a, nsplit)) return ECHO_ESHAPE;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t items = items_of(a);
  if (nsplit <= 1) {
    if (few(a)) hipLaunchKernelGGL(attn_fp8_few_kernel<false>, dim3(items), dim3(64 * FW), 0, st, *a, nullptr, 1);
    else hipLaunchKernelGGL(attn_fp8_kernel<false>, dim3(items), dim3(256), 0, st, *a, nullptr, 1);
  } else {
    if (!ws || ws_bytes < echo_attention_fp8_ws_bytes(a, nsplit) || (uintptr_t)ws % 16) return ECHO_EINVAL;
    if (few(a)) hipLaunchKernelGGL(attn_fp8_few_kernel<true>, dim3(items * nsplit), dim3(64 * FW), 0, st, *a, (float*)ws, nsplit);
    else hipLaunchKernelGGL(attn_fp8_kernel<true>, dim3(items * nsplit), dim3(256), 0, st, *a, (float*)ws, nsplit);
    const int64_t n = (int64_t)a->rows * a->heads * 32 * a->n_q;
    hipLaunchKernelGGL(attn_fp8_join_kernel, dim3((n + 255) / 256), dim3(256), 0, st, *a, (const float*)ws, nsplit);
  }
  ECHO_LAUNCH_CHECK();
  return ECHO_OK;
}

}  // extern "C"
