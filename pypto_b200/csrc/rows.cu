// Rows around a prompt: norm and rotation of query and key heads, quantised rows into the paged caches and back. All of it moves
// each byte once; what bounds the kernels is HBM, or the launch where there are few rows.
#include "rows.cuh"

namespace pto {
namespace {

constexpr int kWarps = 4;  // per block, all three kernels (with eight a block's last warp keeps more registers: 64 tokens 6.2 us for 5.4)
constexpr int kPackedRow = 656;     // 512 int8 | 64 bf16 | 4 f32
constexpr int kPackedNope = 512;
constexpr int kPackedScales = 640;

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Streamed rows: read once, not kept in L1. Not `.nc`: an output may be its input.
__device__ __forceinline__ uint4 ld_row(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack2<T>(u[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// ---- norm and rotation -----------------------------------------------------------------------------------------
// y = x / sqrt(mean x^2 + eps) * w; of the rotated dims every pair (a, b) -> (a cos - b sin, a sin + b cos) with the angle
// position * frequency. A frequency is held in turns a position as a 64-bit binary fraction: the product with the position, taken
// mod 2^64, IS the fraction of a turn, exact at any position, where an angle in fp32 loses 1e-2 rad at 10^5. cos and sin of its
// upper 32 bits are within 2.5e-7, times the amplitude: 9.4e-8 of the fraction's rounding to fp32 (half a step of 2^-24 of half a
// turn), the rest the function's and the amplitude's.
// A lane holds eight neighbouring dims of a head, a power of two of lanes a head, so sums and the other half of a pair travel by
// shuffles. With weights, cosines and sines multiplied beforehand a dim costs four operations besides its conversions: the kernel with a
// norm is bound by instructions (16384 tokens x 40 heads 78 us, issue slots 77 % busy; with the products taken one by one 88, 76 %).
// A warp takes heads of ONE token: its lanes' factors are computed once and stay in registers. With few tokens the heads of one are
// shared out over as many warps as fill the SMs.
template <int kLayout>
__device__ __forceinline__ void rope_lane(uint64_t position, const uint64_t* __restrict__ turns, float amplitude,
                                          int li, int rb, int rv, float (&cs)[8], float (&sn)[8]) {
  // half: dims 8*(li - rb) + e of a half; pairs side by side: pairs 4*(li - rb) + e
  const int first = kLayout == PTO_ROPE_HALF ? 8 * ((li - rb) % (rv / 2)) : 4 * (li - rb);
#pragma unroll
  for (int e = 0; e < (kLayout == PTO_ROPE_HALF ? 8 : 4); ++e) {
    const uint64_t part = position * __ldg(turns + first + e);
    const float half_turns = static_cast<float>(static_cast<int32_t>(part >> 32)) * 4.656612873077392578125e-10f;  // 2^-31
    sincospif(half_turns, &sn[e], &cs[e]);
    cs[e] *= amplitude;
    sn[e] *= amplitude;
  }
}

template <typename T, int kLayout, bool kNorm>
__global__ void __launch_bounds__(kWarps * 32, kNorm ? 6 : 8) norm_rope_kernel(const NormRopeParams p) {
  const int lane = threadIdx.x & 31;
  int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int side = w >= p.side[0].warps ? 1 : 0;
  const NormRopeSide& s = p.side[side];
  if (side == 1) w -= p.side[0].warps;
  if (w >= s.warps) return;
  const int64_t token = w / s.split;
  const int part = static_cast<int>(w - token * s.split);
  const int li = lane & (s.lanes - 1), sub = lane / s.lanes, per = 32 / s.lanes;  // lane of the head, head of the warp, heads a step
  const int vecs = s.d >> 3, rv = p.rotary >> 3, rb = p.rope_last ? vecs - rv : 0;
  const bool rotated = li >= rb && li < rb + rv;
  // where nothing but the rotation is done in place, the other dims stay as they are
  const bool mine = li < vecs && (rotated || !s.rotation_only);
  const T* src = reinterpret_cast<const T*>(s.in) + token * s.in_token + li * 8;
  T* dst = reinterpret_cast<T*>(s.out) + token * s.out_token + li * 8;

  constexpr int kAhead = 4;
  const int steps = (s.heads + per - 1) / per;
  uint4 v[kAhead];
  auto load = [&](int st) {
    const int h = st * per + sub;
    return mine && st < steps && h < s.heads ? ld_row(src + h * s.in_head) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) v[i] = load(part + i * s.split);

  // What a dim is multiplied with and what the pair's other dim is, weights and angles in one; pairs side by side without weights need
  // one of each a pair.
  constexpr bool kHalf = kLayout == PTO_ROPE_HALF;
  constexpr int kEach = kHalf || kNorm ? 8 : 4;
  float mul[kEach], oth[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) mul[e] = 1.f, oth[e] = 0.f;
  const bool second = kHalf && li >= rb + rv / 2;
  const int partner = (lane & ~(s.lanes - 1)) | (rotated ? (second ? li - rv / 2 : li + rv / 2) : li);
  if (rotated) {
    const int64_t pos = p.positions64 ? __ldg(reinterpret_cast<const long long*>(p.positions) + token)
                                      : __ldg(reinterpret_cast<const int*>(p.positions) + token);
    float cs[8], sn[8];
    rope_lane<kLayout>(static_cast<uint64_t>(pos), p.turns, p.amplitude, li, rb, rv, cs, sn);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = kHalf || kEach == 4 ? e : e >> 1;
      mul[e] = cs[i];
      oth[e] = (kHalf ? second : kEach == 4 || (e & 1) != 0) ? sn[i] : -sn[i];
    }
  }
  if (kNorm && li < vecs) {
    float mine_w[8], other_w[8];
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(s.weight) + li), mine_w);
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(s.weight) + (kHalf ? partner & (s.lanes - 1) : li)), other_w);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      mul[e] *= mine_w[e];
      if (rotated) oth[e] *= other_w[kHalf ? e : e ^ 1];
    }
  }
  const float inv_d = 1.f / static_cast<float>(s.d);

  for (int st = part; st < steps; st += kAhead * s.split) {
    // in place the stores of the next steps reach dims that other lanes load: all of them have (at every step 81 us where this has 78)
    if (kLayout == PTO_ROPE_DEINTERLEAVE) __syncwarp();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int now = st + i * s.split;
      if (now >= steps) break;
      float x[8], y[8];
      unpack8<T>(v[i], x);
      v[i] = load(now + kAhead * s.split);
      if constexpr (kEach == 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = kHalf ? __shfl_sync(0xffffffffu, x[e], partner) : x[e ^ 1];
          y[e] = fmaf(x[e], mul[e], other * oth[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = fmaf(x[2 * e], mul[e], -x[2 * e + 1] * oth[e]);
          y[2 * e + 1] = fmaf(x[2 * e + 1], mul[e], x[2 * e] * oth[e]);
        }
      }
      if (kNorm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        for (int o = s.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        // a dim that has no pair takes nothing of its neighbour (inf * 0 is not 0); in halves it is its own, and what an infinity is
        // divided by is one
        if (!kHalf && !rotated && !(ss < INFINITY)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e] * mul[e];
        }
        const float inv = rsqrtf(fmaf(ss, inv_d, p.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= inv;
      }
      const int h = now * per + sub;
      if (!kNorm) {  // a dim that is only copied is copied whatever it is (inf * 0 is not 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = rotated ? y[e] : x[e];
      }
      const bool store = mine && h < s.heads;
      T* out = dst + h * s.out_head;
      if (kLayout != PTO_ROPE_DEINTERLEAVE || !rotated) {
        if (store) *reinterpret_cast<uint4*>(out) = pack8<T>(y);
      } else if (store) {  // the pairs' first values in the first half, their second ones in the second
        T* lo = out - li * 8 + rb * 8 + (li - rb) * 4;
        *reinterpret_cast<uint2*>(lo) = make_uint2(pack2<T>(y[0], y[2]), pack2<T>(y[4], y[6]));
        *reinterpret_cast<uint2*>(lo + rv * 4) = make_uint2(pack2<T>(y[1], y[3]), pack2<T>(y[5], y[7]));
      }
    }
  }
}

// ---- rows into a quantised cache -------------------------------------------------------------------------------
// Per group of 128 dims: up = 127 / max|x|, q = rint(x * up), scale = 1 / up: the prologs' arithmetic, operation by operation. A
// group whose largest magnitude is below 2^-120 (127 / it would leave fp32) is stored as zeros with scale 0; a NaN or an
// infinity makes the scale NaN or infinite, so that the group does not read back as numbers.
// A lane takes 16 dims, eight lanes a group, a warp four groups of one row.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) kv_write_kernel(const KvWriteParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t i = unit / p.chunks;
  const int chunk = static_cast<int>(unit - i * p.chunks);
  if (i >= p.t) return;
  const int64_t row = __ldg(reinterpret_cast<const long long*>(p.index) + i);
  const int g = chunk * 4 + (lane >> 3);
  const bool mine = g < p.groups;
  uint4 a = make_uint4(0, 0, 0, 0), b = a, r = a;
  const T* src = reinterpret_cast<const T*>(p.nope) + i * p.nope_ld + static_cast<int64_t>(chunk) * 512 + lane * 16;
  if (mine) {
    a = ld_row(src);
    b = ld_row(src + 8);
  }
  const bool rope = p.rope != nullptr && chunk == 0 && lane < 8;
  if (rope) r = ld_row(reinterpret_cast<const uint16_t*>(p.rope) + i * p.rope_ld + lane * 8);
  if (row < 0 || row >= p.rows) {
    if (row != -1 && lane == 0) set_status(p.status, PTO_ST_BAD_PAGE, static_cast<int>(row), 70);
    return;
  }
  float x[8], y[8];
  unpack8<T>(a, x);
  unpack8<T>(b, y);
  uint32_t top = 0;  // magnitudes compare as integers, and a NaN is larger than all of them
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float amax = __uint_as_float(top);
  const bool tiny = top < 0x03800000u;  // 2^-120
  const float up = tiny ? 0.f : __fdiv_rn(127.0f, amax);
  const float scale = tiny ? 0.f : __fdiv_rn(1.0f, up);
  uint32_t q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = e < 2 ? x[4 * e + k] : y[4 * (e - 2) + k];
      word |= (static_cast<uint32_t>(__float2int_rn(__fmul_rn(f, up))) & 0xffu) << (8 * k);
    }
    q[e] = word;
  }
  const uint4 qv = make_uint4(q[0], q[1], q[2], q[3]);
  if (p.cache != nullptr) {
    if (mine) {
      *reinterpret_cast<uint4*>(p.cache + row * (static_cast<int64_t>(p.groups) * 128) + chunk * 512 + lane * 16) = qv;
      if ((lane & 7) == 0) {
        const int64_t at = row * p.groups + g;
        if (p.scale_f16) reinterpret_cast<__half*>(p.scales)[at] = __float2half_rn(scale);
        else reinterpret_cast<float*>(p.scales)[at] = scale;
      }
    }
    if (rope) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.rope_cache) + row * 64 + lane * 8) = r;
  }
  if (p.packed != nullptr) {
    int8_t* dst = p.packed + row * kPackedRow;
    *reinterpret_cast<uint4*>(dst + lane * 16) = qv;
    if ((lane & 7) == 0) *reinterpret_cast<float*>(dst + kPackedScales + 4 * g) = scale;
    if (rope) *reinterpret_cast<uint4*>(dst + kPackedNope + lane * 16) = r;
  }
}

// ---- rows back -------------------------------------------------------------------------------------------------
// out[cu[i] + j] = row of position first[i] + j of sequence i. A lane of a warp looks up the cache row of one output row each
// (search of the sequence, block table), then the warp moves its rows, four in flight. Four rows a warp and nine blocks an SM keep more bytes
// on their way than long runs of rows do: 99690 rows in runs of 15, eight in flight 39 us, this 33 (5.5 TB/s).
// int8 -> fp32 without a conversion: 2^23 + (q + 128) is a float whose low byte is q + 128.
__device__ __forceinline__ void dequant16(const uint4& v, float scale, float (&x)[16]) {
  const uint32_t u[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t bits = __byte_perm(u[e >> 2], 0x4b000000u, 0x7540 + (e & 3));
    x[e] = __fmul_rn(__fsub_rn(__uint_as_float(bits), 8388736.0f), scale);
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32, 9) kv_read_kernel(const KvReadParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t base = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * p.per_warp;
  if (base >= p.n) return;
  const int count = static_cast<int>(min(static_cast<int64_t>(p.per_warp), p.n - base));
  // -1: an output row that belongs to no sequence, left as it is; -2: a position without a page, written as zeros
  long long from = -1;
  if (lane < count) {
    const int64_t r = base + lane;
    int lo = 0, hi = p.b;  // sequences that end at or before r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu + mid + 1) <= r) lo = mid + 1;
      else hi = mid;
    }
    if (lo < p.b) {
      const int64_t j = r - __ldg(p.cu + lo);
      if (j >= 0) {
        const int64_t pos = (p.first != nullptr ? static_cast<int64_t>(__ldg(p.first + lo)) : 0) + j;
        from = -2;
        const int64_t blk = pos / p.block_size;
        if (pos >= 0 && blk < p.max_blocks) {
          const int page = __ldg(p.table + static_cast<int64_t>(lo) * p.max_blocks + blk);
          const int64_t at = static_cast<int64_t>(page) * p.block_size + (pos - blk * p.block_size);
          if (page >= 0 && at < p.rows) from = at;
          else set_status(p.status, PTO_ST_BAD_PAGE, page, 71);
        } else {
          set_status(p.status, PTO_ST_BAD_PAGE, static_cast<int>(pos), 72);
        }
      }
    }
  }
  const int64_t width = static_cast<int64_t>(p.groups) * 128;
  constexpr int kAhead = 4;
  for (int chunk = 0; chunk < p.chunks; ++chunk) {
    const int g = chunk * 4 + (lane >> 3);
    const bool mine = g < p.groups;
    for (int r0 = 0; r0 < count; r0 += kAhead) {
      uint4 v[kAhead], rp[kAhead / 4];
      float sc[kAhead];
      long long row[kAhead], rrow[kAhead / 4];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        row[k] = r0 + k < count ? __shfl_sync(0xffffffffu, from, r0 + k) : -1;
        v[k] = make_uint4(0, 0, 0, 0);
        sc[k] = 0.f;
        if (row[k] >= 0 && mine) {
          if (p.packed != nullptr) {
            v[k] = ld_row(p.packed + row[k] * kPackedRow + lane * 16);
            sc[k] = __ldg(reinterpret_cast<const float*>(p.packed + row[k] * kPackedRow + kPackedScales) + g);
          } else {
            v[k] = ld_row(p.cache + row[k] * width + chunk * 512 + lane * 16);
            sc[k] = p.scale_f16 ? __half2float(__ldg(reinterpret_cast<const __half*>(p.scales) + row[k] * p.groups + g))
                                : __ldg(reinterpret_cast<const float*>(p.scales) + row[k] * p.groups + g);
          }
        }
      }
      const bool ropes = p.rope_out != nullptr && chunk == 0;
#pragma unroll
      for (int k = 0; k < kAhead / 4; ++k) {  // the rope part of four rows at once
        const int r = r0 + 4 * k + (lane >> 3);
        rrow[k] = __shfl_sync(0xffffffffu, from, min(r, count - 1));
        if (!ropes || r >= count) rrow[k] = -1;
        rp[k] = make_uint4(0, 0, 0, 0);
        if (rrow[k] >= 0) {
          rp[k] = p.packed != nullptr ? ld_row(p.packed + rrow[k] * kPackedRow + kPackedNope + (lane & 7) * 16)
                                      : ld_row(reinterpret_cast<const uint16_t*>(p.rope) + rrow[k] * 64 + (lane & 7) * 8);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (row[k] == -1 || !mine) continue;
        float x[16];
        dequant16(v[k], sc[k], x);
        if (row[k] < 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 0.f;
        }
        T* dst = reinterpret_cast<T*>(p.out) + (base + r0 + k) * p.out_ld + chunk * 512 + lane * 16;
        __stcs(reinterpret_cast<uint4*>(dst), make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])));
        __stcs(reinterpret_cast<uint4*>(dst) + 1,
               make_uint4(pack2<T>(x[8], x[9]), pack2<T>(x[10], x[11]), pack2<T>(x[12], x[13]), pack2<T>(x[14], x[15])));
      }
#pragma unroll
      for (int k = 0; k < kAhead / 4; ++k) {
        if (rrow[k] == -1) continue;
        const int r = r0 + 4 * k + (lane >> 3);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.rope_out) + (base + r) * p.rope_out_ld + (lane & 7) * 8) = rp[k];
      }
    }
  }
}

template <typename T, bool kNorm>
cudaError_t norm_rope(const NormRopeParams& p, int layout, unsigned grid, cudaStream_t stream) {
  switch (layout) {
    case PTO_ROPE_HALF: norm_rope_kernel<T, PTO_ROPE_HALF, kNorm><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case PTO_ROPE_INTERLEAVED: norm_rope_kernel<T, PTO_ROPE_INTERLEAVED, kNorm><<<grid, kWarps * 32, 0, stream>>>(p); break;
    default: norm_rope_kernel<T, PTO_ROPE_DEINTERLEAVE, kNorm><<<grid, kWarps * 32, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace

// Warps of a side: heads of a token go to one warp when tokens alone fill the SMs, to several otherwise.
void norm_rope_plan(NormRopeSide* s, int64_t t, int num_sms) {
  s->lanes = 1;
  while (s->lanes * 8 < s->d) s->lanes *= 2;
  const int per = 32 / s->lanes, steps = (s->heads + per - 1) / per;
  const int64_t fill = static_cast<int64_t>(num_sms) * 32;
  int64_t split = (fill + t - 1) / t;
  if (split > steps) split = steps;
  if (split < 1) split = 1;
  s->split = static_cast<int>(split);
  s->warps = s->heads > 0 ? t * split : 0;
}

cudaError_t launch_norm_rope(const NormRopeParams& p, int dtype, int layout, cudaStream_t stream) {
  if (p.side[0].warps > 0 && p.side[1].warps > 0 && (p.side[0].weight == nullptr) != (p.side[1].weight == nullptr)) {
    for (int i = 0; i < 2; ++i) {  // a kernel with a norm and one without
      NormRopeParams one = p;
      one.side[0] = p.side[i];
      one.side[1].warps = 0;
      one.side[1].weight = nullptr;
      const cudaError_t e = launch_norm_rope(one, dtype, layout, stream);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }
  const int64_t warps = p.side[0].warps + p.side[1].warps;
  if (warps == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  const bool norm = p.side[0].weight != nullptr || p.side[1].weight != nullptr;
  count_launch();
  if (dtype == PTO_DT_BF16) return norm ? norm_rope<__nv_bfloat16, true>(p, layout, grid, stream) : norm_rope<__nv_bfloat16, false>(p, layout, grid, stream);
  return norm ? norm_rope<__half, true>(p, layout, grid, stream) : norm_rope<__half, false>(p, layout, grid, stream);
}

cudaError_t launch_kv_write(const KvWriteParams& p, int dtype, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(p.t) * p.chunks + kWarps - 1) / kWarps);
  count_launch();
  if (dtype == PTO_DT_BF16) kv_write_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(p);
  else kv_write_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv_read(KvReadParams p, int dtype, int num_sms, cudaStream_t stream) {
  // rows a warp: one while there are fewer rows than warps in flight, then up to four, which share one look-up
  const int64_t fill = static_cast<int64_t>(num_sms) * 48;
  int64_t per = (p.n + fill - 1) / fill;
  per = per > 4 ? 4 : per;
  p.per_warp = static_cast<int>(per);
  const int64_t warps = (p.n + per - 1) / per;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  count_launch();
  if (dtype == PTO_DT_BF16) kv_read_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(p);
  else kv_read_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace pto
