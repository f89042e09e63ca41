// Rotary position embedding of a chunk's queries and keys, dense or on the way
// into the paged cache.
//
// A row x of head_dim d with rotary width R turns, for each frequency i < R/2,
// the pair (a, b) = (x_i, x_{i + R/2}) -- or (x_{2i}, x_{2i+1}) -- by the angle
// position * inv_freq_i:
//   a' = a c - b s,  b' = b c + a s,  (c, s) = factor (cos, sin)(angle);
// elements from R on stay. With several position axes (time, height, width of
// an image's tokens) frequency i takes the position of axis axis_of[i].
//
// The angle is formed and reduced in fp64: at position 10^6 the fp32 product is
// off by up to 0.03 rad, and the fp64 one, in turns, by 2^-53 of some 10^5
// turns. What is left of a turn, in fp32, goes to fp32 sin and cos, and what that rounding
// leaves (up to 2^-26 turns, as much as the rounding of sin and cos) to their first-order terms;
// the products are fp32, and each result is rounded once.
#include <type_traits>

#include "spv_common.h"

using namespace spv;

namespace {

constexpr double kInvTwoPi = 0.15915494309189533576888;

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

// A pair turned by t = (c, s), with the same roundings in every kernel.
__device__ __forceinline__ float2 turned(float a, float b, float2 t) {
  return make_float2(fmaf(a, t.x, -(b * t.y)), fmaf(b, t.x, a * t.y));
}

// cos and sin of position * inv_freq_i, times the factor.
__device__ __forceinline__ float2 turn_of(const RotaryParams& p, int b, int j, int i) {
  const int axis = p.axis_of ? min(max(p.axis_of[i], 0), p.axes - 1) : 0;
  const int pos = p.positions ? p.positions[((size_t)axis * p.B + b) * p.C + j] : p.start[b] + j;
  const double turns = p.inv_freq[i] * kInvTwoPi;
  const double r = fma((double)pos, turns, -__builtin_rint((double)pos * turns));  // in [-1/2, 1/2]
  const float f = (float)r, rest = (float)(r - f) * 6.283185307f;  // what f leaves, in radians
  float s, c;
  sincospif(2.f * f, &s, &c);
  return make_float2(fmaf(-s, rest, c) * p.factor, fmaf(c, rest, s) * p.factor);
}

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

// One thread per element pair (or element past the rotary width) of a row; one
// workgroup per (entry, token). Any head_dim, stride and alignment.
template <int DT, int KO, bool APPEND>
__global__ __launch_bounds__(256) void rotary_elem_kernel(RotaryParams p) {
  const int b = blockIdx.x / p.C, j = blockIdx.x - b * p.C;
  const int half = p.R / 2, items = half + (p.d - p.R);
  int row = -1;
  if constexpr (APPEND) {
    if (p.plan_in) {
      row = p.plan_in[(size_t)b * p.C + j];
    } else {
      int n;
      row = pool_row(p, b, j, &n);
      if (threadIdx.x == 0) {
        if (p.plan_out) p.plan_out[(size_t)b * p.C + j] = row;
        if (j == 0 && n > 0) {
          const int sid = p.seq_ids[b], end = p.start[b] + n;
          if (p.seq_lens[sid] < end) p.seq_lens[sid] = end;
        }
      }
    }
  }
  const int blk = row >= 0 ? row / p.bs : 0, off = row >= 0 ? row - blk * p.bs : 0;
  for (int it = threadIdx.x; it < (p.Hq + p.Hkv) * items; it += blockDim.x) {
    const int hh = it / items, i = it - hh * items;
    const bool isq = hh < p.Hq;
    const int h = isq ? hh : hh - p.Hq;
    const uint8_t* src = isq ? p.q : p.k;
    if (!src) continue;
    const long long* st = isq ? p.qs : p.ks;
    const size_t in = (size_t)((long long)b * st[0] + (long long)j * st[1] + (long long)h * st[2]);
    size_t out;
    if (isq) out = (size_t)((long long)b * p.qos[0] + (long long)j * p.qos[1] + (long long)h * p.qos[2]);
    else if constexpr (APPEND) out = ((((size_t)p.layer * p.cap + blk) * p.Hkv + h) * p.bs + off) * p.d;
    else out = (size_t)((long long)b * p.kos[0] + (long long)j * p.kos[1] + (long long)h * p.kos[2]);
    if (APPEND && !isq && row < 0) continue;
    auto put = [&](int e, float x) {
      if (isq) store_elem<DT>(p.q_out, out + e, x);
      else if constexpr (APPEND) store_elem<DT>(p.kpool, out + e, x);
      else store_elem<KO>(p.k_out, out + e, x);
    };
    if (i < half) {
      const int e0 = p.interleaved ? 2 * i : i, e1 = p.interleaved ? 2 * i + 1 : i + half;
      const float a = load_elem<DT>(src, in + e0), c = load_elem<DT>(src, in + e1);
      const float2 t = turn_of(p, b, j, i);
      const float2 y = turned(a, c, t);
      put(e0, y.x);
      put(e1, y.y);
    } else {
      const int e = p.R + (i - half);
      put(e, load_elem<DT>(src, in + e));
    }
  }
  if constexpr (APPEND) {
    if (row < 0) return;
    for (int it = threadIdx.x; it < p.Hkv * p.d; it += blockDim.x) {
      const int h = it / p.d, e = it - h * p.d;
      const size_t in = (size_t)((long long)b * p.vs[0] + (long long)j * p.vs[1] + (long long)h * p.vs[2]) + e;
      const size_t out = ((((size_t)p.layer * p.cap + blk) * p.Hkv + h) * p.d + e) * p.bs + off;
      if constexpr (DT == SPV_F32) reinterpret_cast<uint32_t*>(p.vpool)[out] = reinterpret_cast<const uint32_t*>(p.v)[in];
      else reinterpret_cast<uint16_t*>(p.vpool)[out] = reinterpret_cast<const uint16_t*>(p.v)[in];
    }
  }
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

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

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
    return w;
  }
};

// Host-chosen shape of the launch.
struct VecShape {
  int TT, items, hs, hpw, slices, tiles;  // tokens, pieces per row, heads at once, heads per slice, slices, tiles of C
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

template <int DT, bool APPEND>
__global__ __launch_bounds__(kVecThreads) void rotary_vec_kernel(RotaryParams p, VecShape v) {
  constexpr int ES = DT == SPV_F32 ? 4 : 2, E = 16 / ES;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int s_row[kMaxTT];
  const int x = blockIdx.x, slice = blockIdx.y;
  const int b = x / v.tiles, tile = x - b * v.tiles;
  if (APPEND && slice >= v.slices) {
    copy_values<DT, APPEND>(p, b, tile, slice - v.slices, lds);
    return;
  }
  const int j0 = tile * v.TT, nt = min(v.TT, p.C - j0);
  if (nt <= 0) return;
  const int c = threadIdx.x % v.items, rest = threadIdx.x / v.items, t = rest % v.TT, hs = rest / v.TT;
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
  };
  for (int h = h0; h < end; h += v.hs) {
    put(h);
    if (h + v.hs < end) load(h + v.hs);
  }
}

size_t vec_lds(const RotaryParams& p, const VecShape& v, int es, bool append) {
  const size_t turns = (size_t)v.TT * (p.R / 2) * sizeof(float2), values = append ? (size_t)kVT * p.d * es : 0;
  return turns > values ? turns : values;
}

// Whether the vector kernel takes the call: whole 16-byte pieces that begin on
// 16-byte addresses, and rows short enough for one workgroup's threads.
bool vec_shape(const RotaryParams& p, int es, bool append, VecShape& v) {
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
  if (v.items > kVecThreads) return false;
  v.TT = 1;
  while (v.TT < kMaxTT && v.TT < p.C && 2 * v.TT * v.items <= kVecThreads) v.TT *= 2;
  v.hs = kVecThreads / (v.items * v.TT);
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
  return (long long)p.B * v.tiles <= (1LL << 23) && v.slices + p.Hkv <= 65535 && vec_lds(p, v, es, append) <= 65536;
}

// Shapes and frequencies common to both entry points.
bool rotary_args_ok(int dtype, int32_t B, int32_t C, int32_t hq, int32_t hkv, int32_t d, int32_t rotary_dim,
                    int32_t axes, int32_t interleaved, const double* inv_freq, const int32_t* axis_of) {
  if (dtype != SPV_F32 && dtype != SPV_BF16 && dtype != SPV_F16) return false;
  if (B < 0 || C < 1 || hq < 0 || hkv < 0 || hq > 65535 || hkv > 65535 || d < 1 || d > 65536 || rotary_dim < 0 ||
      rotary_dim > d || rotary_dim % 2 || axes < 1 || (interleaved != 0 && interleaved != 1))
    return false;
  if (rotary_dim > 0 && (!inv_freq || (axes > 1 && !axis_of))) return false;
  return (long long)B * C <= (1LL << 23);  // one workgroup of 256 threads per token at most
}

template <bool APPEND>
void launch_vec(const RotaryParams& p, const VecShape& v, int dtype, hipStream_t s) {
  const size_t smem = vec_lds(p, v, dtype_size(dtype), APPEND);
  const dim3 grid((unsigned)(p.B * v.tiles), (unsigned)(v.slices + (APPEND ? p.Hkv : 0))), blk(kVecThreads);
#define SPV_VEC(DT) hipLaunchKernelGGL((rotary_vec_kernel<DT, APPEND>), grid, blk, smem, s, p, v)
  if (dtype == SPV_F32) SPV_VEC(SPV_F32);
  else if (dtype == SPV_BF16) SPV_VEC(SPV_BF16);
  else SPV_VEC(SPV_F16);
#undef SPV_VEC
}

void set_strides(long long* dst, const int64_t* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}

}  // namespace

extern "C" {

int spv_rotary(void* q_out, const void* q, void* k_out, const void* k, int dtype, int k_out_dtype,
               const int64_t* strides, const int32_t* positions, const double* inv_freq, const int32_t* axis_of,
               int32_t axes, float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
               int32_t head_dim, int32_t rotary_dim, int32_t interleaved, void* stream) {
  if (!strides || !positions || (!q && !k) || (q && !q_out) || (k && !k_out)) return SPV_ERR_ARG;
  if ((q && num_q_heads < 1) || (k && num_kv_heads < 1)) return SPV_ERR_ARG;
  if (!rotary_args_ok(dtype, B, C, num_q_heads, num_kv_heads, head_dim, rotary_dim, axes, interleaved, inv_freq,
                      axis_of))
    return SPV_ERR_ARG;
  if (k_out_dtype != dtype && k_out_dtype != SPV_F32) return SPV_ERR_ARG;
  if (B == 0) return SPV_OK;
  RotaryParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.k = static_cast<const uint8_t*>(k);
  p.q_out = static_cast<uint8_t*>(q_out);
  p.k_out = static_cast<uint8_t*>(k_out);
  set_strides(p.qos, strides);
  set_strides(p.qs, strides + 3);
  set_strides(p.kos, strides + 6);
  set_strides(p.ks, strides + 9);
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.axis_of = axes > 1 ? axis_of : nullptr;
  p.factor = factor;
  p.B = B;
  p.C = C;
  p.Hq = q ? num_q_heads : 0;
  p.Hkv = k ? num_kv_heads : 0;
  p.d = head_dim;
  p.R = rotary_dim;
  p.interleaved = interleaved;
  p.axes = axes;
  hipStream_t s = (hipStream_t)stream;
  VecShape v;
  if (k_out_dtype == dtype && vec_shape(p, dtype_size(dtype), false, v)) {
    launch_vec<false>(p, v, dtype, s);
    SPV_CHECK_LAUNCH();
    return SPV_OK;
  }
  const dim3 grid((unsigned)(B * C)), blk(256);
#define SPV_ROT(DT, KO) hipLaunchKernelGGL((rotary_elem_kernel<DT, KO, false>), grid, blk, 0, s, p)
  if (dtype == SPV_F32) SPV_ROT(SPV_F32, SPV_F32);
  else if (dtype == SPV_BF16 && k_out_dtype == SPV_BF16) SPV_ROT(SPV_BF16, SPV_BF16);
  else if (dtype == SPV_BF16) SPV_ROT(SPV_BF16, SPV_F32);
  else if (k_out_dtype == SPV_F16) SPV_ROT(SPV_F16, SPV_F16);
  else SPV_ROT(SPV_F16, SPV_F32);
#undef SPV_ROT
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

int spv_kv_rotary_append(void* q_out, const void* q, const void* k_new, const void* v_new, int dtype,
                         const int64_t* strides, void* k_pool, void* v_pool, int32_t* block_tables,
                         int32_t max_blocks_per_seq, int32_t* num_blocks, int32_t* seq_lens, int32_t* free_stack,
                         int32_t* free_flag, int32_t* ctr, const int32_t* seq_ids, const int32_t* start_pos,
                         const int32_t* positions, const double* inv_freq, const int32_t* axis_of, int32_t axes,
                         float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
                         int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int32_t layer, int32_t capacity,
                         int32_t block_size, int32_t may_alloc, int32_t follow_plan, int32_t* write_plan,
                         void* stream) {
  if (!strides || !k_new || !v_new || (q && !q_out) || !k_pool || !v_pool || !block_tables || !num_blocks ||
      !seq_lens || !ctr || !seq_ids || !start_pos || (follow_plan && (!write_plan || may_alloc)))
    return SPV_ERR_ARG;
  if ((q && num_q_heads < 1) || num_kv_heads < 1 || layer < 0 || capacity < 1 || block_size < 1 ||
      max_blocks_per_seq < 1)
    return SPV_ERR_ARG;
  if (!rotary_args_ok(dtype, B, C, num_q_heads, num_kv_heads, head_dim, rotary_dim, axes, interleaved, inv_freq,
                      axis_of))
    return SPV_ERR_ARG;
  if ((long long)capacity * block_size > 0x7fffffffLL) return SPV_ERR_ARG;  // pool rows are int32
  if (!positions && axes != 1) return SPV_ERR_ARG;
  if (may_alloc && (!free_stack || !free_flag)) return SPV_ERR_ARG;
  if (B == 0) return SPV_OK;
  if (may_alloc) {
    const int rc = spv_kv_append(k_pool, v_pool, dtype, nullptr, nullptr, block_tables, max_blocks_per_seq,
                                 num_blocks, seq_lens, free_stack, free_flag, ctr, seq_ids, start_pos, B, C, layer,
                                 capacity, block_size, num_kv_heads, head_dim, 1, -1, stream);
    if (rc != SPV_OK) return rc;
  }
  RotaryParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.k = static_cast<const uint8_t*>(k_new);
  p.v = static_cast<const uint8_t*>(v_new);
  p.q_out = static_cast<uint8_t*>(q_out);
  p.kpool = static_cast<uint8_t*>(k_pool);
  p.vpool = static_cast<uint8_t*>(v_pool);
  set_strides(p.qos, strides);
  set_strides(p.qs, strides + 3);
  set_strides(p.ks, strides + 6);
  set_strides(p.vs, strides + 9);
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.axis_of = axes > 1 ? axis_of : nullptr;
  p.factor = factor;
  p.tables = block_tables;
  p.nblocks = num_blocks;
  p.seq_lens = seq_lens;
  p.seq_ids = seq_ids;
  p.start = start_pos;
  p.ctr = ctr;
  p.plan_out = follow_plan ? nullptr : write_plan;
  p.plan_in = follow_plan ? write_plan : nullptr;
  p.B = B;
  p.C = C;
  p.Hq = q ? num_q_heads : 0;
  p.Hkv = num_kv_heads;
  p.d = head_dim;
  p.R = rotary_dim;
  p.interleaved = interleaved;
  p.axes = axes;
  p.maxb = max_blocks_per_seq;
  p.layer = layer;
  p.cap = capacity;
  p.bs = block_size;
  hipStream_t s = (hipStream_t)stream;
  VecShape v;
  if (vec_shape(p, dtype_size(dtype), true, v)) {
    launch_vec<true>(p, v, dtype, s);
    SPV_CHECK_LAUNCH();
    return SPV_OK;
  }
  const dim3 grid((unsigned)(B * C)), blk(256);
#define SPV_ROT(DT) hipLaunchKernelGGL((rotary_elem_kernel<DT, DT, true>), grid, blk, 0, s, p)
  if (dtype == SPV_F32) SPV_ROT(SPV_F32);
  else if (dtype == SPV_BF16) SPV_ROT(SPV_BF16);
  else SPV_ROT(SPV_F16);
#undef SPV_ROT
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // extern "C"
