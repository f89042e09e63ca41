// What the rotary kernels share: the turn of a frequency at a position, a pair
// turned by it, the 16-byte pieces that rows travel in, and the body of a launch
// over rows of whole pieces.
#pragma once

#include <type_traits>

#include "spv_common.h"

namespace spv {

constexpr double kInvTwoPi = 0.15915494309189533576888;

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// A pair turned by t = (c, s), with the same roundings in every kernel.
__device__ __forceinline__ float2 turned(float a, float b, float2 t) {
  return make_float2(fmaf(a, t.x, -(b * t.y)), fmaf(b, t.x, a * t.y));
}

// cos and sin of position * inv_freq_i, times the factor, for token j of entry b
// (positions: (axes, B, C), or null: start + token on every axis; axis_of: null
// for axis 0).
template <class P>
__device__ __forceinline__ float2 turn_of(const P& p, int b, int j, int i) {
  const int axis = p.axis_of ? min(max(p.axis_of[i], 0), p.axes - 1) : 0;
  const int pos = p.positions ? p.positions[((size_t)axis * p.B + b) * p.C + j] : p.start[b] + j;
  const double turns = p.inv_freq[i] * kInvTwoPi;
  const double r = fma((double)pos, turns, -__builtin_rint((double)pos * turns));  // in [-1/2, 1/2]
  const float f = (float)r, rest = (float)(r - f) * 6.283185307f;  // what f leaves, in radians
  float s, c;
  sincospif(2.f * f, &s, &c);
  return make_float2(fmaf(-s, rest, c) * p.factor, fmaf(c, rest, s) * p.factor);
}

// What a row of d elements with this sum of squares is multiplied by:
// 1 / sqrt(mean of squares + eps), in fp32.
__device__ __forceinline__ float norm_factor(float sum_sq, int d, float eps) {
  return 1.f / sqrtf(sum_sq / (float)d + eps);
}

template <int DT>
struct Piece {  // 16 bytes as fp32
  static constexpr int E = DT == SPV_F32 ? 4 : 8;
  float x[E];
  __device__ __forceinline__ void unpack(u32x4_t w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SPV_F32) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == SPV_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const uint32_t word = w[i];  // a bit cast of the vector's element itself takes element 0
        const f16x2_t h = __builtin_bit_cast(f16x2_t, word);
        x[2 * i] = (float)h[0];
        x[2 * i + 1] = (float)h[1];
      }
    }
  }
  __device__ __forceinline__ u32x4_t pack() const {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SPV_F32) w[i] = __float_as_uint(x[i]);
      else if constexpr (DT == SPV_BF16)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x[2 * i], x[2 * i + 1]}, bf16x2_t));
      else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x[2 * i], x[2 * i + 1]}, f16x2_t));
    }
    // The compiler (clang of ROCm 7.2) has given the registers of the first words away where a vector
    // built word by word met another one behind a branch: it takes this one as written at once.
    asm("" : "+v"(w));
    return w;
  }
};

struct RotaryParams {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* q_out;
  uint8_t* k_out;  // dense (spv_rotary)
  uint8_t* kpool;  // paged (spv_kv_rotary_append)
  uint8_t* vpool;
  long long qs[3], ks[3], vs[3], qos[3], kos[3];  // element strides: batch, token, head
  const int32_t* positions;  // (axes, B, C), or null: start + token on every axis
  const double* inv_freq;    // R / 2
  const int32_t* axis_of;    // R / 2, or null: axis 0
  float factor;
  const float* wq;  // NORM: d weights of the query heads, and of the key heads (null: 1)
  const float* wk;
  float eps;
  const int32_t* tables;
  const int32_t* nblocks;
  int32_t* seq_lens;
  const int32_t* seq_ids;
  const int32_t* start;
  const int32_t* ctr;
  int32_t* plan_out;       // record the chunk's pool rows here (or null)
  const int32_t* plan_in;  // follow these pool rows (or null)
  int B, C, Hq, Hkv, d, R, interleaved, axes, maxb, layer, cap, bs;
};

// The pool row (block * block_size + offset) of chunk token j of entry b, or -1
// where the append writes nothing: past the sequence an exhausted pool cut off,
// past its blocks, or a block id outside the pool -- the rule of spv_kv_append
// with write_limit_b = -1.
__device__ __forceinline__ int pool_row(const RotaryParams& p, int b, int j, int* valid) {
  const int sid = p.seq_ids[b], s0 = p.start[b];
  const int ex = p.ctr[CTR_EXHAUSTED];
  const int n = (s0 < 0 || (ex && b > ex - 1)) ? 0 : min(p.C, p.nblocks[sid] * p.bs - s0);
  *valid = n;
  if (j >= n) return -1;
  const int at = s0 + j;
  const int phys = p.tables[(size_t)sid * p.maxb + min(at / p.bs, p.maxb - 1)];
  return (unsigned)phys < (unsigned)p.cap ? phys * p.bs + at % p.bs : -1;
}

// Rows of whole 16-byte pieces. A workgroup takes TT tokens of one entry and a
// slice of the heads. A thread keeps one token and one piece pair (the pieces
// that rotate with each other; past the rotary width one piece) and goes over
// the slice's heads with it; the waves of a CU keep enough loads in flight (four
// heads ahead per thread and 16 tokens a workgroup took 18.4 us over the 75.5 MB
// below). The turns of the
// workgroup's tokens are computed once, into LDS, while the first rows travel.
// The slices behind the query and key heads copy the values, one (16 positions,
// head) each, transposed through LDS so that whole pages are stored as 16-byte
// pieces.
// What bounds it: the rows' bytes, each read and written once, for prompts (75.5 MB of
// bf16 queries and keys in 15.0 us, 5.0 TB/s; with the values and the cache's writes 30.7 MB
// a layer in 9.0); a few dependent round trips (start, table, length, position) for decode
// chunks (8 tokens 3.9 us, 32 chunks of 6 tokens 4.5).
constexpr int kVecThreads = 256;
constexpr int kMaxTT = 8;
constexpr int kVT = 16;  // positions of a value tile

// Host-chosen shape of the launch.
struct VecShape {
  // tokens, pieces per row, threads per row (NORM: a power of two), heads at once, heads per slice, slices, tiles of C
  int TT, items, lanes, hs, hpw, slices, tiles;
};

template <int DT, bool APPEND>
__device__ __forceinline__ void copy_values(const RotaryParams& p, int b, int tile, int h, uint8_t* lds) {
  using T = typename std::conditional<DT == SPV_F32, uint32_t, uint16_t>::type;
  constexpr int ES = sizeof(T), E = 16 / ES;
  __shared__ int s_row[kVT];
  const int s0 = p.start[b], first = (s0 >= 0 ? s0 / kVT * kVT : s0) + tile * kVT;  // the tile's positions
  const int j0 = max(first - s0, 0), nt = min(p.C, first + kVT - s0) - j0;           // its chunk tokens
  if (nt <= 0) return;
  const int vec = p.d / E;
  T* const sv = reinterpret_cast<T*>(lds);  // [token][d]
  const uint8_t* src = p.v + ((long long)b * p.vs[0] + (long long)j0 * p.vs[1] + (long long)h * p.vs[2]) * ES;
  for (int i = threadIdx.x; i < nt * vec; i += kVecThreads) {
    const int t = i / vec, c = i - t * vec;
    reinterpret_cast<u32x4_t*>(sv)[i] = *reinterpret_cast<const u32x4_t*>(src + (long long)t * p.vs[1] * ES + 16 * c);
  }
  if ((int)threadIdx.x < nt) {
    int n;
    s_row[threadIdx.x] = p.plan_in ? p.plan_in[(size_t)b * p.C + j0 + threadIdx.x] : pool_row(p, b, j0 + threadIdx.x, &n);
  }
  __syncthreads();
  T* const pool = reinterpret_cast<T*>(p.vpool) + ((size_t)p.layer * p.cap * p.Hkv + h) * (size_t)p.d * p.bs;
  const size_t step = (size_t)p.Hkv * p.d * p.bs;  // elements from a block's page to the next block's
  if (nt == kVT && p.bs % kVT == 0 && s_row[0] >= 0 && s_row[kVT - 1] == s_row[0] + kVT - 1) {
    // 16 tokens side by side in one page: 16-byte pieces of each dim's row
    const int blk = s_row[0] / p.bs, off = s_row[0] - blk * p.bs;  // a multiple of 16, as the first position is
    T* const dst = pool + blk * step + off;
    constexpr int kPer = kVT / E;
    for (int i = threadIdx.x; i < p.d * kPer; i += kVecThreads) {
      const int e = i / kPer, q = i - e * kPer;
      u32x4_t w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (ES == 4) w[k] = sv[(q * E + k) * p.d + e];
        else w[k] = sv[(q * E + 2 * k) * p.d + e] | (uint32_t)sv[(q * E + 2 * k + 1) * p.d + e] << 16;
      }
      *reinterpret_cast<u32x4_t*>(dst + (size_t)e * p.bs + q * E) = w;
    }
    return;
  }
  for (int i = threadIdx.x; i < nt * p.d; i += kVecThreads) {
    const int e = i / nt, t = i - e * nt, row = s_row[t];  // tokens fastest: neighbours of a dim's row
    if (row < 0) continue;
    const int blk = row / p.bs, off = row - blk * p.bs;
    pool[blk * step + (size_t)e * p.bs + off] = sv[t * p.d + e];
  }
}

// Workgroup (x, slice) of the launch; lds: vec_lds() bytes.
template <int DT, bool APPEND, bool NORM>
__device__ __forceinline__ void rotary_vec_rows(const RotaryParams& p, const VecShape& v, int x, int slice,
                                                uint8_t* lds) {
  constexpr int ES = DT == SPV_F32 ? 4 : 2, E = 16 / ES;
  __shared__ int s_row[kMaxTT];
  const int b = x / v.tiles, tile = x - b * v.tiles;
  if (APPEND && slice >= v.slices) {
    copy_values<DT, APPEND>(p, b, tile, slice - v.slices, lds);
    return;
  }
  const int j0 = tile * v.TT, nt = min(v.TT, p.C - j0);
  if (nt <= 0) return;
  const int lane = threadIdx.x % v.lanes, rest = threadIdx.x / v.lanes, t = rest % v.TT, hs = rest / v.TT;
  const int c = NORM ? min(lane, v.items - 1) : lane;
  const int half = p.R / 2, n2 = half / E;  // frequencies, piece pairs of a row
  const bool pair = c < n2;
  const int c0 = !pair ? 2 * n2 + (c - n2) : p.interleaved ? 2 * c : c;  // the thread's pieces of a row
  const int c1 = !pair ? c0 : p.interleaved ? 2 * c + 1 : c + n2;
  const int H = p.Hq + p.Hkv, end = min((slice + 1) * v.hpw, H);
  const bool mine = t < nt && hs < v.hs;
  const int j = j0 + min(t, nt - 1);
  const uint8_t* const qrow = p.q + ((long long)b * p.qs[0] + (long long)j * p.qs[1]) * ES;
  const uint8_t* const krow = p.k + ((long long)b * p.ks[0] + (long long)j * p.ks[1]) * ES;
  u32x4_t in0{}, in1{};
  auto load = [&](int h) {
    const uint8_t* row = h < p.Hq ? qrow + (long long)h * p.qs[2] * ES : krow + (long long)(h - p.Hq) * p.ks[2] * ES;
    in0 = *reinterpret_cast<const u32x4_t*>(row + 16 * c0);
    in1 = *reinterpret_cast<const u32x4_t*>(row + 16 * c1);
  };
  const int h0 = slice * v.hpw + hs;
  if (mine && h0 < end) load(h0);
  if constexpr (APPEND) {
    if ((int)threadIdx.x < nt && (slice == 0 || end > p.Hq)) {
      const int jj = j0 + threadIdx.x;
      int row;
      if (p.plan_in) {
        row = p.plan_in[(size_t)b * p.C + jj];
      } else {
        int n;
        row = pool_row(p, b, jj, &n);
        if (slice == 0) {
          if (p.plan_out) p.plan_out[(size_t)b * p.C + jj] = row;
          if (jj == 0 && n > 0) {
            const int sid = p.seq_ids[b], upto = p.start[b] + n;
            if (p.seq_lens[sid] < upto) p.seq_lens[sid] = upto;
          }
        }
      }
      s_row[threadIdx.x] = row;
    }
  }
  float2* const turns = reinterpret_cast<float2*>(lds);  // [token][frequency]
  for (int i = threadIdx.x; i < nt * half; i += kVecThreads) {
    const int tt = i / half, f = i - tt * half;
    turns[i] = turn_of(p, b, j0 + tt, f);
  }
  float* const weights = reinterpret_cast<float*>(turns + v.TT * half);  // NORM: [queries | keys][d]
  if constexpr (NORM) {
    for (int i = threadIdx.x; i < 2 * p.d; i += kVecThreads) {
      const float* const w = i < p.d ? p.wq : p.wk;
      weights[i] = w ? w[i < p.d ? i : i - p.d] : 1.f;
    }
  }
  __syncthreads();
  if (!mine) return;
  int blk = 0, off = 0, row = -1;
  if constexpr (APPEND) {
    if (end > p.Hq) {
      row = s_row[t];
      if (row >= 0) {
        blk = row / p.bs;
        off = row - blk * p.bs;
      }
    }
  }
  // Where the rows go: chosen by values, for a choice between the arguments' addresses becomes a
  // load from one of them for every head.
  const long long qstep = p.qos[2] * ES, kstep = APPEND ? (long long)p.bs * p.d * ES : p.kos[2] * ES;
  uint8_t* const qdst = p.q_out + ((long long)b * p.qos[0] + (long long)j * p.qos[1]) * ES;
  uint8_t* const kdst =
      APPEND ? p.kpool + ((((size_t)p.layer * p.cap + blk) * p.Hkv) * p.bs + off) * (size_t)(p.d * ES)
             : p.k_out + ((long long)b * p.kos[0] + (long long)j * p.kos[1]) * ES;
  auto put = [&](int h) {
    if (APPEND && h >= p.Hq && row < 0) return;
    uint8_t* const out = h < p.Hq ? qdst + h * qstep : kdst + (h - p.Hq) * kstep;
    if constexpr (!NORM) {
      // One pair of stores for both ways, past the rotary width of the one piece twice: 75.5 MB of queries and keys in
      // 15.3 us, with a store apart for such pieces 16.4 (where half of each row turns, 16.2 and 15.6).
      u32x4_t y0 = in0, y1 = in1;  // past the rotary width both are the one piece
      if (pair) {
        Piece<DT> a, d;
        a.unpack(y0);
        d.unpack(y1);
        const float2* const tc = turns + t * half + c * E;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          // neighbours: pairs within a piece, the first half of them in the first
          if (p.interleaved) {
            float* const z = i < E / 2 ? &a.x[2 * i] : &d.x[2 * i - E];
            const float2 y = turned(z[0], z[1], tc[i]);
            z[0] = y.x;
            z[1] = y.y;
          } else {
            const float2 y = turned(a.x[i], d.x[i], tc[i]);
            a.x[i] = y.x;
            d.x[i] = y.y;
          }
        }
        y0 = a.pack();
        y1 = d.pack();
      }
      *reinterpret_cast<u32x4_t*>(out + 16 * c0) = y0;
      *reinterpret_cast<u32x4_t*>(out + 16 * c1) = y1;
      return;
    }
    Piece<DT> a, d;
    a.unpack(in0);
    d.unpack(in1);
    if constexpr (NORM) {  // the row's threads are neighbours in one wave
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(a.x[i], a.x[i], ss);
      if (pair) {
#pragma unroll
        for (int i = 0; i < E; ++i) ss = fmaf(d.x[i], d.x[i], ss);
      }
      if (lane >= v.items) ss = 0.f;
      for (int o = v.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
      if (lane >= v.items) return;
      const float inv = norm_factor(ss, p.d, p.eps);
      const float* const w = weights + (h < p.Hq ? 0 : p.d);
#pragma unroll
      for (int i = 0; i < E; ++i) a.x[i] *= inv * w[c0 * E + i];
      if (!pair) {
        *reinterpret_cast<u32x4_t*>(out + 16 * c0) = a.pack();
        return;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) d.x[i] *= inv * w[c1 * E + i];
    }
    const float2* const tc = turns + t * half + c * E;
    if (p.interleaved) {  // neighbours: pairs within a piece, the first half of them in the first
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float* const z = i < E / 2 ? &a.x[2 * i] : &d.x[2 * i - E];
        const float2 y = turned(z[0], z[1], tc[i]);
        z[0] = y.x;
        z[1] = y.y;
      }
      *reinterpret_cast<u32x4_t*>(out + 16 * c0) = a.pack();
      *reinterpret_cast<u32x4_t*>(out + 16 * c1) = d.pack();
      return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float2 y = turned(a.x[i], d.x[i], tc[i]);
      a.x[i] = y.x;
      d.x[i] = y.y;
    }
    *reinterpret_cast<u32x4_t*>(out + 16 * c0) = a.pack();
    *reinterpret_cast<u32x4_t*>(out + 16 * c1) = d.pack();
  };
  for (int h = h0; h < end; h += v.hs) {
    put(h);
    if (h + v.hs < end) load(h + v.hs);
  }
}

inline size_t vec_lds(const RotaryParams& p, const VecShape& v, int es, bool append, bool norm) {
  const size_t turns = (size_t)v.TT * (p.R / 2) * sizeof(float2) + (norm ? 2 * (size_t)p.d * sizeof(float) : 0);
  const size_t values = append ? (size_t)kVT * p.d * es : 0;
  return turns > values ? turns : values;
}

// Whether the vector kernel takes the call: whole 16-byte pieces that begin on
// 16-byte addresses, and rows short enough for one workgroup's threads (NORM: one wave's).
inline bool vec_shape(const RotaryParams& p, int es, bool append, bool norm, VecShape& v) {
  const int E = 16 / es;
  if (p.d % E || p.R % (2 * E)) return false;
  auto aligned = [&](const void* ptr, const long long* st) {
    if (!ptr) return true;
    return (uintptr_t)ptr % 16 == 0 && st[0] * es % 16 == 0 && st[1] * es % 16 == 0 && st[2] * es % 16 == 0;
  };
  if (!aligned(p.q, p.qs) || !aligned(p.q_out, p.qos) || !aligned(p.k, p.ks)) return false;
  if (append ? !aligned(p.v, p.vs) || (uintptr_t)p.kpool % 16 || (uintptr_t)p.vpool % 16 : !aligned(p.k_out, p.kos))
    return false;
  v.items = p.R / (2 * E) + (p.d - p.R) / E;
  if (v.items > (norm ? 64 : kVecThreads)) return false;
  v.lanes = v.items;
  if (norm)
    for (v.lanes = 1; v.lanes < v.items;) v.lanes *= 2;
  v.TT = 1;
  while (v.TT < kMaxTT && v.TT < p.C && 2 * v.TT * v.lanes <= kVecThreads) v.TT *= 2;
  v.hs = kVecThreads / (v.lanes * v.TT);
  const int H = p.Hq + p.Hkv;
  v.tiles = (p.C + v.TT - 1) / v.TT;
  // Slices of the heads until there are about 1,024 workgroups, each thread with one head at least.
  const long long wgs = (long long)p.B * v.tiles, want = (1024 + wgs - 1) / wgs;
  const int most = (H + v.hs - 1) / v.hs;
  const int ns = (int)(want < most ? want : most);
  v.hpw = ((H + ns - 1) / ns + v.hs - 1) / v.hs * v.hs;
  v.slices = (H + v.hpw - 1) / v.hpw;
  if (append) {  // value tiles: the chunk's positions by sixteens from a multiple of sixteen
    const int vt = (p.C + kVT - 1) / kVT + 1;
    if (vt > v.tiles) v.tiles = vt;
  }
  return (long long)p.B * v.tiles <= (1LL << 23) && v.slices + p.Hkv <= 65535 && vec_lds(p, v, es, append, norm) <= 65536;
}

// A launch of the dense rows of p (rotary.hip), any shape and alignment.
int rotary_queries(const RotaryParams& p, int dtype, bool norm, hipStream_t s);

}  // namespace spv
