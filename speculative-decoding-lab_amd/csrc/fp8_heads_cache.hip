// Writing and reading an 8-bit paged cache with a scale for each (block, head).
//
// Write: for the rows x of a chunk that fall into a block, per kv head and
// separately for K and V,
//   a = max |x| (finite x),  s' = max(s, a / 448),
//   q = e4m3(x / s') (0 where s' = 0),  and, where s' > s, q = e4m3((q s) / s')
// for every other row of the block's page. With TURN the keys are rotated first
// (with NORM normed before that, rotary_common.h) and quantised unrounded, and the
// queries go through the same launch. Products and quotients are correctly rounded
// fp32. What is not finite is stored as NaN and left out of a.
//
// Read: x = q * s in fp32, rounded once to the output's type.
#include "fp8_heads.h"

using namespace spv;

namespace {

constexpr int kThreads = 256, kMaxThreads = 1024;
constexpr int kRowLanes = 16;                    // threads of a row while it is turned
constexpr int kPad = 16;                         // floats: a wave's four rows on banks of their own

struct HeadWrite {
  RotaryParams r;  // keys, values, pools and tables
  RotaryParams q;  // the queries alone (Hkv = 0)
  float* scales;
  int T, tile, limit_b;  // blocks an entry's chunk touches at most; rows staged at once (at most)
  unsigned nkv;          // workgroups of keys and values, before those of the queries
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}

// One workgroup per (entry, block that the chunk touches, kv head); behind them
// the queries' workgroups of rotary_vec_rows.
// VEC (16-byte rows, head_dim and blocks of whole 16, a chunk's rows in a block staged at once): 16 bytes of the page per
// thread and turn, K's dims or V's tokens; of a block that is not wholly new they are asked for before the rows are turned.
// Byte by byte, prompts of 4 x 3,001 tokens with two kv heads of 128 took 21.4 us (now 11.9), 32 verify chunks of 6
// tokens 9.8 (now 8.9).
// What bounds it: round trips one behind the other (start, then tables, rows and turns, then scales and the page, 3 us
// together for verify chunks), the norm and rotation of a row by 16 threads (1.8), quotients and stores (1.5); prompts
// read their rows meanwhile (18.9 MB moved, 3.8 us at the rate of a large copy).
template <int IT, bool TURN, bool NORM, bool QUERY, bool VEC>
__global__ __launch_bounds__(VEC ? kMaxThreads : kThreads) void head_write_kernel(HeadWrite w, VecShape v) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ float s_red[2][kMaxThreads / 64];
  const int threads = VEC ? blockDim.x : kThreads;
  if constexpr (QUERY) {
    if (blockIdx.x >= w.nkv) {
      if (VEC && threadIdx.x >= kVecThreads) return;  // whole waves: barriers do without them
      const int x = blockIdx.x - w.nkv, per = w.q.B * v.tiles;
      rotary_vec_rows<IT, false, NORM>(w.q, v, x % per, x / per, lds);
      return;
    }
  }
  const RotaryParams& p = w.r;
  const int h = blockIdx.x % p.Hkv, bt = blockIdx.x / p.Hkv, b = bt / w.T, t = bt - b * w.T;
  const int s0 = p.start[b];
  if (s0 < 0) return;
  const int blk = s0 / p.bs + t;
  const int lo = max(s0 - blk * p.bs, 0), hi_c = min(s0 + p.C - blk * p.bs, p.bs);
  if (hi_c <= lo) return;
  const int sid = p.seq_ids[b], d = p.d, st = d + kPad, half = p.R / 2;
  // VEC: the first 16 bytes of K and V per thread are on their way while tables and turns are looked up.
  constexpr int E = Piece<IT>::E;
  const int row_pieces = d / E;
  [[maybe_unused]] u32x4_t raw_k{}, raw_v{};
  auto piece_of = [&](const uint8_t* x, const long long (&s)[3], int i) {
    const int r = i / row_pieces, at = (i - r * row_pieces) * E, j = blk * p.bs + lo - s0 + r;
    const long long o = (long long)b * s[0] + (long long)j * s[1] + (long long)h * s[2] + at;
    return *reinterpret_cast<const u32x4_t*>(x + o * (16 / E));
  };
  if constexpr (VEC) {
    if ((int)threadIdx.x < (hi_c - lo) * row_pieces) {
      raw_k = piece_of(p.k, p.ks, threadIdx.x);
      raw_v = piece_of(p.v, p.vs, threadIdx.x);
    }
  }
  int limit = w.limit_b;
  if (limit < 0) {
    const int ex = p.ctr[CTR_EXHAUSTED];
    limit = ex ? ex - 1 : 0x7fffffff;
  }
  const int n = b > limit ? 0 : min(p.C, p.nblocks[sid] * p.bs - s0);
  const int phys = p.tables[(size_t)sid * p.maxb + min(blk, p.maxb - 1)];
  float* const sk = reinterpret_cast<float*>(lds);
  float* const sv = sk + (size_t)w.tile * st;
  float2* const turns = reinterpret_cast<float2*>(sv + (size_t)w.tile * st);
  if constexpr (VEC && TURN) {
    for (int i = threadIdx.x; i < (hi_c - lo) * half; i += threads) {
      const int r = i / half, f = i - r * half;
      turns[i] = turn_of(p, b, blk * p.bs + lo - s0 + r, f);
    }
  }
  float* const weights = reinterpret_cast<float*>(turns + (size_t)w.tile * half);  // VEC and NORM: of a row
  if constexpr (VEC && NORM) {
    if (p.wk)
      for (int i = threadIdx.x; i < d; i += threads) weights[i] = p.wk[i];
  }
  const int hi = min(hi_c, s0 + n - blk * p.bs);
  if (n <= 0 || hi <= lo || blk >= p.maxb || (unsigned)phys >= (unsigned)p.cap) return;  // never outside the pool
  if (t == 0 && h == 0 && threadIdx.x == 0 && p.seq_lens[sid] < s0 + n) p.seq_lens[sid] = s0 + n;

  float* const page_scale = w.scales + scale_of(p.layer, p.cap, phys, p.Hkv, h);
  const float old_k = page_scale[0], old_v = page_scale[1];
  const size_t page = page_of(p.layer, p.cap, phys, p.Hkv, h, p.bs, d);
  uint8_t* const kp = p.kpool + page;  // [token][d]
  uint8_t* const vp = p.vpool + page;  // [d][token]
  const int pieces = p.bs * d / 16;    // VEC: of a page; V's come first
  [[maybe_unused]] u32x4_t held{};
  auto codes_at = [&](int i) { return reinterpret_cast<u32x4_t*>(i < pieces ? vp : kp) + (i < pieces ? i : i - pieces); };
  if constexpr (VEC) {
    if (hi - lo < p.bs && (int)threadIdx.x < 2 * pieces) held = *codes_at(threadIdx.x);
  }

  // Rows [ra, rb) of the block into LDS, the keys normed and turned.
  float ak = 0.f, av = 0.f;
  auto finite_abs = [](float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
  };
  auto stage = [&](int ra, int rb) {
    const int j0 = blk * p.bs + ra - s0, rows = rb - ra;
    if constexpr (VEC) {
      for (int i = threadIdx.x; i < rows * row_pieces; i += threads) {
        if (i != (int)threadIdx.x) {
          raw_k = piece_of(p.k, p.ks, i);
          raw_v = piece_of(p.v, p.vs, i);
        }
        const int r = i / row_pieces, e = (i - r * row_pieces) * E;
        Piece<IT> x, y;
        x.unpack(raw_k);
        y.unpack(raw_v);
#pragma unroll
        for (int q = 0; q < E; q += 4) {
          *reinterpret_cast<float4*>(sk + r * st + e + q) = make_float4(x.x[q], x.x[q + 1], x.x[q + 2], x.x[q + 3]);
          *reinterpret_cast<float4*>(sv + r * st + e + q) = make_float4(y.x[q], y.x[q + 1], y.x[q + 2], y.x[q + 3]);
        }
#pragma unroll
        for (int q = 0; q < E; ++q) {
          if constexpr (!TURN) ak = fmaxf(ak, finite_abs(x.x[q]));
          av = fmaxf(av, finite_abs(y.x[q]));
        }
      }
    }
    for (int i = VEC ? rows * d : threadIdx.x; i < rows * d; i += threads) {
      const int r = i / d, e = i - r * d;
      const long long at = (long long)b * p.ks[0] + (long long)(j0 + r) * p.ks[1] + (long long)h * p.ks[2] + e;
      const long long av_at = (long long)b * p.vs[0] + (long long)(j0 + r) * p.vs[1] + (long long)h * p.vs[2] + e;
      const float xk = load_elem<IT>(p.k, (size_t)at), xv = load_elem<IT>(p.v, (size_t)av_at);
      sk[r * st + e] = xk;
      sv[r * st + e] = xv;
      if constexpr (!TURN) ak = fmaxf(ak, finite_abs(xk));
      av = fmaxf(av, finite_abs(xv));
    }
    if constexpr (TURN && !VEC) {
      for (int i = threadIdx.x; i < rows * half; i += threads) {
        const int r = i / half, f = i - r * half;
        turns[i] = turn_of(p, b, j0 + r, f);
      }
    }
    __syncthreads();
    if constexpr (TURN) {
      const int lane = threadIdx.x % kRowLanes;
      for (int r = threadIdx.x / kRowLanes; r < rows; r += threads / kRowLanes) {
        float* const x = sk + r * st;
        if constexpr (NORM) {
          float ss = 0.f;
          for (int e = lane; e < d; e += kRowLanes) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int o = kRowLanes / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
          const float inv = norm_factor(ss, d, p.eps);
          for (int e = lane; e < d; e += kRowLanes) x[e] *= p.wk ? inv * (VEC ? weights : p.wk)[e] : inv;
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        for (int i = lane; i < half; i += kRowLanes) {
          const int e0 = p.interleaved ? 2 * i : i, e1 = p.interleaved ? 2 * i + 1 : i + half;
          const float2 y = turned(x[e0], x[e1], turns[r * half + i]);
          x[e0] = y.x;
          x[e1] = y.y;
          ak = fmaxf(ak, fmaxf(finite_abs(y.x), finite_abs(y.y)));
        }
        for (int e = p.R + lane; e < d; e += kRowLanes) ak = fmaxf(ak, finite_abs(x[e]));
      }
      __syncthreads();
    }
  };
  // Tiles of the block's rows; one that holds them all is staged once.
  const int t0 = VEC ? 0 : lo / w.tile, t1 = VEC ? 0 : (hi - 1) / w.tile;
  auto first = [&](int k) { return VEC ? lo : max(lo, k * w.tile); };
  auto last = [&](int k) { return VEC ? hi : min(hi, (k + 1) * w.tile); };
  for (int k = t0; k <= t1; ++k) {
    if (k > t0) __syncthreads();
    stage(first(k), last(k));
  }
  ak = wave_max(ak);
  av = wave_max(av);
  if ((threadIdx.x & 63) == 0) {
    s_red[0][threadIdx.x >> 6] = ak;
    s_red[1][threadIdx.x >> 6] = av;
  }
  __syncthreads();
  float a0 = 0.f, a1 = 0.f;
  for (int i = 0; i < threads / 64; ++i) {
    a0 = fmaxf(a0, s_red[0][i]);
    a1 = fmaxf(a1, s_red[1][i]);
  }
  const float nk = fmaxf(old_k, __fdiv_rn(a0, 448.f)), nv = fmaxf(old_v, __fdiv_rn(a1, 448.f));
  if (VEC && usual_scale(nk) && usual_scale(nv)) {
    const float yk = __fdiv_rn(1.f, nk), yv = __fdiv_rn(1.f, nv);
    for (int i = threadIdx.x; i < 2 * pieces; i += threads) {
      const bool is_v = i < pieces;
      const float scale = is_v ? nv : nk, y = is_v ? yv : yk, old = is_v ? old_v : old_k;
      const int at = (is_v ? i : i - pieces) * 16, line = is_v ? p.bs : d, e = at / line, c0 = at - e * line;
      // V: tokens c0 .. c0 + 15 of dim e; K: dims c0 .. c0 + 15 of token e. Bytes [from, to) of them are new.
      const int from = is_v ? max(lo - c0, 0) : 0, to = is_v ? min(hi - c0, 16) : e >= lo && e < hi ? 16 : 0;
      const bool again = scale > old;  // for the others
      if (to <= from && !again) continue;
      u32x4_t w = held;
      if (from > 0 || to < 16) {
        if (i != (int)threadIdx.x) w = *codes_at(i);
        if (again) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float x[4];
            decode4(w[q], x);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = quotient(__fmul_rn(x[k], old), scale, y);
            w[q] = encode4(x);
          }
        }
      }
      if (to > from) {
        const float* const x0 = is_v ? sv + (c0 - lo) * st + e : sk + (e - lo) * st + c0;
        const int step = is_v ? st : 1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = quotient(x0[min(max(4 * q + k, from), to - 1) * step], scale, y);
          const int a = min(max(from - 4 * q, 0), 4), b = min(max(to - 4 * q, 0), 4);
          const uint32_t in = (uint32_t)((1ull << (8 * b)) - 1) & ~(uint32_t)((1ull << (8 * a)) - 1);
          w[q] = (w[q] & ~in) | (encode4(x) & in);
        }
      }
      *codes_at(i) = w;
    }
    if (threadIdx.x == 0) {
      page_scale[0] = nk;
      page_scale[1] = nv;
    }
    return;
  }
  for (int k = t0; k <= t1; ++k) {
    const int ra = first(k), rb = last(k), rows = rb - ra;
    if (t1 > t0) {
      __syncthreads();
      stage(ra, rb);
    }
    for (int i = threadIdx.x; i < rows * d; i += threads) {
      const int r = i / d, e = i - r * d;
      kp[(size_t)(ra + r) * d + e] = encode1(quotient(sk[r * st + e], nk));
    }
    for (int i = threadIdx.x; i < rows * d; i += threads) {
      const int e = i / rows, r = i - e * rows;
      vp[(size_t)e * p.bs + ra + r] = encode1(quotient(sv[r * st + e], nv));
    }
  }
  const int others = (p.bs - (hi - lo)) * d;
  if (nk > old_k || nv > old_v) {
    for (int i = threadIdx.x; i < others; i += threads) {
      int r = i / d;
      const int e = i - r * d;
      if (r >= lo) r += hi - lo;
      if (nk > old_k) {
        uint8_t* const q = kp + (size_t)r * d + e;
        *q = encode1(requotient(fp8e4m3_to_f32(*q), old_k, nk));
      }
      if (nv > old_v) {
        uint8_t* const q = vp + (size_t)e * p.bs + r;
        *q = encode1(requotient(fp8e4m3_to_f32(*q), old_v, nv));
      }
    }
  }
  if (threadIdx.x == 0) {
    page_scale[0] = nk;
    page_scale[1] = nv;
  }
}

struct HeadRead {
  const uint8_t* kpool;
  const uint8_t* vpool;
  const float* scales;
  const int32_t* table;
  void* out;
  int length, layer, cap, bs, hkv, d;
};

// out[0][p][h][e] = K, out[1][p][h][e] = V of positions p < length.
template <int OT>
__global__ __launch_bounds__(kThreads) void head_read_kernel(HeadRead p) {
  const size_t per_tok = (size_t)p.hkv * p.d, total = (size_t)p.length * per_tok;
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
    const int pos = (int)(i / per_tok), rest = (int)(i - (size_t)pos * per_tok);
    const int h = rest / p.d, e = rest - h * p.d, blk = pos / p.bs, off = pos - blk * p.bs;
    const int id = p.table[blk], phys = (unsigned)id < (unsigned)p.cap ? id : 0;
    const float* const s = p.scales + scale_of(p.layer, p.cap, phys, p.hkv, h);
    const size_t page = page_of(p.layer, p.cap, phys, p.hkv, h, p.bs, p.d);
    store_elem<OT>(p.out, i, fp8e4m3_to_f32(p.kpool[page + (size_t)off * p.d + e]) * s[0]);
    store_elem<OT>(p.out, total + i, fp8e4m3_to_f32(p.vpool[page + (size_t)e * p.bs + off]) * s[1]);
  }
}

// The same in pieces: a workgroup takes kReadTokens positions of a head, K (4 codes per thread and turn) or V, whose
// page has a dim's tokens side by side (4 x 4 codes, put across in registers). Bound by the bytes it stores and by the
// table, scale and page one behind the other: 32,768 positions of two heads of 64 to bf16 (25.2 MB, floor 5.1 us) in 7.8
// us, 3.2 TB/s; code by code 20.8.
constexpr int kReadTokens = 64;
template <int OT>
__global__ __launch_bounds__(kThreads) void head_read_vec_kernel(HeadRead p) {
  const int t0 = blockIdx.x * kReadTokens, h = blockIdx.y, d = p.d, lines = min(kReadTokens, p.length - t0);
  const size_t step = (size_t)p.hkv * d, total = (size_t)p.length * step;
  auto page_at = [&](int pos, int& off, size_t& page) {
    const int blk = pos / p.bs, id = p.table[blk], phys = (unsigned)id < (unsigned)p.cap ? id : 0;
    off = pos - blk * p.bs;
    page = page_of(p.layer, p.cap, phys, p.hkv, h, p.bs, d);
    return p.scales + scale_of(p.layer, p.cap, phys, p.hkv, h);
  };
  auto store4 = [&](size_t at, const float* x) {
    if constexpr (OT == SPV_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      u32x2_t w;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (OT == SPV_BF16)
          w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x[2 * i], x[2 * i + 1]}, bf16x2_t));
        else
          w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x[2 * i], x[2 * i + 1]}, f16x2_t));
      }
      asm("" : "+v"(w));
      *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + at) = w;
    }
  };
  int off;
  size_t page;
  float x[4];
  if (blockIdx.z == 0) {
    for (int i = threadIdx.x; i < lines * (d / 4); i += kThreads) {
      const int t = i / (d / 4), e = (i - t * (d / 4)) * 4;
      const float s = page_at(t0 + t, off, page)[0];
      decode4(*reinterpret_cast<const uint32_t*>(p.kpool + page + (size_t)off * d + e), x);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= s;
      store4((size_t)(t0 + t) * step + (size_t)h * d + e, x);
    }
  } else {
    for (int i = threadIdx.x; i < (lines + 3) / 4 * (d / 4); i += kThreads) {
      const int t = i / (d / 4) * 4, e = (i - t / 4 * (d / 4)) * 4;
      const float s = page_at(t0 + t, off, page)[1];
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = *reinterpret_cast<const uint32_t*>(p.vpool + page + (size_t)(e + q) * p.bs + off);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t + j >= lines) break;
        const uint32_t sel = 0x0c0c0400u + 0x0101u * j;  // byte j of the second operand, then of the first
        const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], sel), hi = __builtin_amdgcn_perm(w[3], w[2], sel);
        decode4(lo | hi << 16, x);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] *= s;
        store4(total + (size_t)(t0 + t + j) * step + (size_t)h * d + e, x);
      }
    }
  }
}

constexpr size_t kLdsBytes = 65536;
constexpr size_t kVecLdsBytes = 158720;  // VEC: of 160 KiB, with what the kernel has beside it

// LDS of a key / value workgroup that stages `rows` rows at once.
size_t write_lds(int rows, int d, int R, bool turn) {
  return (size_t)rows * (2 * (d + kPad) * sizeof(float) + (turn ? R / 2 * sizeof(float2) : 0));
}

// Rows staged at once: the whole block's, or as many as fit (a multiple of 16); 0: none fit.
int write_tile(int bs, int d, int R, bool turn) {
  int rows = bs;
  while (rows > 16 && write_lds(rows, d, R, turn) > kLdsBytes) rows = (rows / 2 + 15) / 16 * 16;
  while (rows > 1 && write_lds(rows, d, R, turn) > kLdsBytes) rows /= 2;
  return write_lds(rows, d, R, turn) <= kLdsBytes ? rows : 0;
}

template <int IT, bool VEC>
void launch_write(const HeadWrite& w, const VecShape& v, bool turn, bool norm, bool query, unsigned grid, int threads,
                  size_t smem, hipStream_t s) {
#define SPV_W(TURN, NORM, QUERY)                                                                                \
  do {                                                                                                          \
    if (smem > 65536)                                                                                           \
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&head_write_kernel<IT, TURN, NORM, QUERY, VEC>),  \
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);                         \
    hipLaunchKernelGGL((head_write_kernel<IT, TURN, NORM, QUERY, VEC>), dim3(grid), dim3(threads), smem, s, w,  \
                       v);                                                                                      \
  } while (0)
  if (!turn) SPV_W(false, false, false);
  else if (!norm && !query) SPV_W(true, false, false);
  else if (!norm) SPV_W(true, false, true);
  else if (!query) SPV_W(true, true, false);
  else SPV_W(true, true, true);
#undef SPV_W
}

struct PoolArgs {  // the append's pool arguments, as every append takes them
  void* k_pool;
  void* v_pool;
  float* scales;
  int32_t* tables;
  int32_t maxb;
  int32_t* nblocks;
  int32_t* seq_lens;
  int32_t* free_stack;
  int32_t* free_flag;
  int32_t* ctr;
  const int32_t* seq_ids;
  const int32_t* start;
};

bool shape_ok(const PoolArgs& a, int dtype, int32_t B, int32_t C, int32_t layer, int32_t num_layers, int32_t cap,
              int32_t bs, int32_t hkv, int32_t d) {
  return a.k_pool && a.v_pool && a.scales && a.tables && a.nblocks && a.seq_lens && a.seq_ids && a.start &&
         (dtype == SPV_F32 || dtype == SPV_BF16 || dtype == SPV_F16) && B >= 0 && C >= 1 && layer >= 0 &&
         num_layers >= 1 && layer < num_layers && cap >= 1 && bs >= 1 && hkv >= 1 && hkv <= 65535 && d >= 1 &&
         a.maxb >= 1 && (long long)num_layers * hkv <= 0x7fffffffLL;
}

// The missing blocks of the chunk, with zero scales in every layer and head.
int allocate(const PoolArgs& a, int32_t B, int32_t C, int32_t num_layers, int32_t cap, int32_t bs, int32_t hkv,
             int32_t d, void* stream) {
  return spv_kv_append_fp8(a.k_pool, a.v_pool, a.scales, SPV_F32, nullptr, nullptr, a.tables, a.maxb, a.nblocks,
                           a.seq_lens, a.free_stack, a.free_flag, a.ctr, a.seq_ids, a.start, B, C, 0,
                           num_layers * hkv, cap, bs, hkv, d, 1, -1, stream);
}

// What a write launches.
struct WriteShape {
  unsigned grid;
  int threads;
  size_t smem;
  bool vec, query;  // query: the queries are turned in the same launch
  VecShape v;
};

// The shape of a write of w.r, whose pools are a's, or an error: found before anything is allocated, so that a call
// which is refused changes nothing.
int write_shape(HeadWrite& w, const PoolArgs& a, int dtype, bool turn, bool norm, int32_t limit_b, WriteShape& x) {
  RotaryParams& p = w.r;
  p.kpool = static_cast<uint8_t*>(a.k_pool);
  p.vpool = static_cast<uint8_t*>(a.v_pool);
  p.tables = a.tables;
  p.nblocks = a.nblocks;
  p.seq_lens = a.seq_lens;
  p.seq_ids = a.seq_ids;
  p.start = a.start;
  p.ctr = a.ctr;
  p.maxb = a.maxb;
  w.scales = a.scales;
  w.limit_b = limit_b;
  if ((long long)p.bs * p.d > (1LL << 30)) return SPV_ERR_ARG;  // a page is counted in 32 bits
  const long long blocks = ((long long)p.C + p.bs - 2) / p.bs + 1, entries = blocks * p.B;
  if (entries > 0x3fffffffLL) return SPV_ERR_ARG;
  w.T = (int)blocks;
  w.tile = write_tile(p.bs, p.d, p.R, turn);
  if (!w.tile) return SPV_ERR_UNSUPPORTED;
  if (p.B == 0) return SPV_OK;  // nothing to launch
  const long long nkv = entries * p.Hkv;
  x.smem = write_lds(w.tile, p.d, p.R, turn);
  size_t query_smem = 0;
  long long grid = nkv;
  if (p.q) {
    w.q = p;
    w.q.Hkv = 0;
    w.q.k = nullptr;
    x.query = vec_shape(w.q, dtype_size(dtype), false, norm, x.v);
    if (x.query) {
      query_smem = vec_lds(w.q, x.v, dtype_size(dtype), false, norm);
      if (query_smem > x.smem) x.smem = query_smem;
      grid += (long long)p.B * x.v.tiles * x.v.slices;
    }
  }
  // vec: the rows of a chunk in a block at once, and the weights
  const int rows = p.bs < p.C ? p.bs : p.C;
  size_t vec_smem = write_lds(rows, p.d, p.R, turn) + (norm ? p.d * sizeof(float) : 0);
  if (vec_smem < query_smem) vec_smem = query_smem;
  x.vec = vec_smem <= kVecLdsBytes && p.d % 16 == 0 && p.bs % 16 == 0 &&
          (((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.kpool | (uintptr_t)p.vpool) & 15) == 0;
  for (int i = 0; i < 3; ++i)
    x.vec = x.vec && (p.ks[i] * dtype_size(dtype)) % 16 == 0 && (p.vs[i] * dtype_size(dtype)) % 16 == 0;
  x.threads = kThreads;
  if (x.vec) {
    w.tile = rows;
    x.smem = vec_smem;
    // A thread for eight elements: 8 chunks of 71 fp32 tokens into blocks of 64, head_dim 128, take 17.2 us a call, with
    // 256 threads 26.9 (a workgroup has a CU to itself there).
    while (x.threads < kMaxThreads && x.threads * 8 < rows * p.d) x.threads *= 2;
  }
  if (grid * x.threads > 0xffffffffLL) return SPV_ERR_ARG;  // a launch counts its threads in 32 bits
  w.nkv = (unsigned)nkv;
  x.grid = (unsigned)grid;
  return SPV_OK;
}

int write(const HeadWrite& w, const WriteShape& x, int dtype, bool turn, bool norm, hipStream_t s) {
#define SPV_W(IT)                                                                                       \
  x.vec ? launch_write<IT, true>(w, x.v, turn, norm, x.query, x.grid, x.threads, x.smem, s)             \
        : launch_write<IT, false>(w, x.v, turn, norm, x.query, x.grid, x.threads, x.smem, s)
  if (dtype == SPV_F32) SPV_W(SPV_F32);
  else if (dtype == SPV_BF16) SPV_W(SPV_BF16);
  else SPV_W(SPV_F16);
#undef SPV_W
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

void strides3(long long* dst, const int64_t* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}

}  // namespace

extern "C" {

int spv_kv_append_fp8_heads(void* k_pool, void* v_pool, float* kv_scales, int new_dtype, const void* k_new,
                            const void* v_new, const int64_t* strides, int32_t* block_tables,
                            int32_t max_blocks_per_seq, int32_t* num_blocks, int32_t* seq_lens, int32_t* free_stack,
                            int32_t* free_flag, int32_t* ctr, const int32_t* seq_ids, const int32_t* start_pos,
                            int32_t B, int32_t C, int32_t layer, int32_t num_layers, int32_t capacity,
                            int32_t block_size, int32_t num_kv_heads, int32_t head_dim, int32_t may_alloc,
                            int32_t write_limit_b, void* stream) {
  const PoolArgs a{k_pool, v_pool, kv_scales, block_tables, max_blocks_per_seq, num_blocks, seq_lens, free_stack,
                   free_flag, ctr, seq_ids, start_pos};
  const bool alloc_only = !k_new && !v_new;
  if (!shape_ok(a, alloc_only ? SPV_F32 : new_dtype, B, C, layer, num_layers, capacity, block_size, num_kv_heads,
                head_dim))
    return SPV_ERR_ARG;
  if (!alloc_only && (!k_new || !v_new || !strides)) return SPV_ERR_ARG;
  if (write_limit_b < -1 || write_limit_b > B || (write_limit_b < 0 && !ctr)) return SPV_ERR_ARG;
  if (may_alloc && (!free_stack || !free_flag || !ctr)) return SPV_ERR_ARG;
  HeadWrite w{};
  WriteShape x{};
  if (!alloc_only) {
    RotaryParams& p = w.r;
    p.k = static_cast<const uint8_t*>(k_new);
    p.v = static_cast<const uint8_t*>(v_new);
    strides3(p.ks, strides);
    strides3(p.vs, strides + 3);
    p.B = B;
    p.C = C;
    p.Hkv = num_kv_heads;
    p.d = head_dim;
    p.layer = layer;
    p.cap = capacity;
    p.bs = block_size;
    const int rc = write_shape(w, a, new_dtype, false, false, write_limit_b, x);
    if (rc != SPV_OK) return rc;
  }
  if (B == 0) return SPV_OK;
  if (may_alloc) {
    const int rc = allocate(a, B, C, num_layers, capacity, block_size, num_kv_heads, head_dim, stream);
    if (rc != SPV_OK) return rc;
  }
  return alloc_only ? SPV_OK : write(w, x, new_dtype, false, false, (hipStream_t)stream);
}

int spv_kv_rotary_append_fp8_heads(void* q_out, const void* q, const void* k_new, const void* v_new, int dtype,
                                   const int64_t* strides, int32_t normed, const float* q_weight,
                                   const float* k_weight, float eps, void* k_pool, void* v_pool, float* kv_scales,
                                   int32_t* block_tables, int32_t max_blocks_per_seq, int32_t* num_blocks,
                                   int32_t* seq_lens, int32_t* free_stack, int32_t* free_flag, int32_t* ctr,
                                   const int32_t* seq_ids, const int32_t* start_pos, const int32_t* positions,
                                   const double* inv_freq, const int32_t* axis_of, int32_t axes, float factor,
                                   int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                   int32_t rotary_dim, int32_t interleaved, int32_t layer, int32_t num_layers,
                                   int32_t capacity, int32_t block_size, int32_t may_alloc, void* stream) {
  const PoolArgs a{k_pool, v_pool, kv_scales, block_tables, max_blocks_per_seq, num_blocks, seq_lens, free_stack,
                   free_flag, ctr, seq_ids, start_pos};
  if (!shape_ok(a, dtype, B, C, layer, num_layers, capacity, block_size, num_kv_heads, head_dim)) return SPV_ERR_ARG;
  if (!strides || !k_new || !v_new || !ctr || (q && (!q_out || num_q_heads < 1 || num_q_heads > 65535)))
    return SPV_ERR_ARG;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 || axes < 1 || (!positions && axes != 1) ||
      (interleaved != 0 && interleaved != 1) || (rotary_dim > 0 && (!inv_freq || (axes > 1 && !axis_of))))
    return SPV_ERR_ARG;
  if (normed && !(eps >= 0.f && eps < 1e30f)) return SPV_ERR_ARG;
  if (may_alloc && (!free_stack || !free_flag)) return SPV_ERR_ARG;
  if ((long long)B * C > (1LL << 23)) return SPV_ERR_ARG;
  HeadWrite w{};
  RotaryParams& p = w.r;
  p.q = static_cast<const uint8_t*>(q);
  p.k = static_cast<const uint8_t*>(k_new);
  p.v = static_cast<const uint8_t*>(v_new);
  p.q_out = static_cast<uint8_t*>(q_out);
  strides3(p.qos, strides);
  strides3(p.qs, strides + 3);
  strides3(p.ks, strides + 6);
  strides3(p.vs, strides + 9);
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.axis_of = axes > 1 ? axis_of : nullptr;
  p.factor = factor;
  p.wq = q_weight;
  p.wk = k_weight;
  p.eps = eps;
  p.B = B;
  p.C = C;
  p.Hq = q ? num_q_heads : 0;
  p.Hkv = num_kv_heads;
  p.d = head_dim;
  p.R = rotary_dim;
  p.interleaved = interleaved;
  p.axes = axes;
  p.layer = layer;
  p.cap = capacity;
  p.bs = block_size;
  WriteShape x{};
  int rc = write_shape(w, a, dtype, true, normed != 0, -1, x);
  if (rc != SPV_OK || B == 0) return rc;
  if (may_alloc) {
    rc = allocate(a, B, C, num_layers, capacity, block_size, num_kv_heads, head_dim, stream);
    if (rc != SPV_OK) return rc;
  }
  rc = write(w, x, dtype, true, normed != 0, (hipStream_t)stream);
  if (rc != SPV_OK || !q || x.query) return rc;
  return rotary_queries(w.q, dtype, normed != 0, (hipStream_t)stream);
}

int spv_kv_gather_fp8_heads(const void* k_pool, const void* v_pool, const float* kv_scales,
                            const int32_t* block_tables, int32_t max_blocks_per_seq, int32_t seq_id, int32_t length,
                            int32_t layer, int32_t capacity, int32_t block_size, int32_t num_kv_heads,
                            int32_t head_dim, void* out, int out_dtype, void* stream) {
  if (!k_pool || !v_pool || !kv_scales || !block_tables || !out || seq_id < 0 || length < 0 || layer < 0 ||
      capacity < 1 || block_size < 1 || num_kv_heads < 1 || head_dim < 1 ||
      (out_dtype != SPV_F32 && out_dtype != SPV_BF16 && out_dtype != SPV_F16))
    return SPV_ERR_ARG;
  if ((length + (long long)block_size - 1) / block_size > max_blocks_per_seq) return SPV_ERR_ARG;
  if ((long long)num_kv_heads * head_dim > 0x7fffffffLL) return SPV_ERR_ARG;
  if (length == 0) return SPV_OK;
  const HeadRead p{static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), kv_scales,
                   block_tables + (size_t)seq_id * max_blocks_per_seq, out, length, layer, capacity, block_size,
                   num_kv_heads, head_dim};
  hipStream_t s = (hipStream_t)stream;
  if (head_dim % 4 == 0 && block_size % 4 == 0 && num_kv_heads <= 65535 && (uintptr_t)out % 16 == 0 &&
      ((uintptr_t)k_pool | (uintptr_t)v_pool) % 4 == 0) {
    const dim3 grid((unsigned)((length + (long long)kReadTokens - 1) / kReadTokens), (unsigned)num_kv_heads, 2), blk(kThreads);
    if (out_dtype == SPV_F32) hipLaunchKernelGGL(head_read_vec_kernel<SPV_F32>, grid, blk, 0, s, p);
    else if (out_dtype == SPV_BF16) hipLaunchKernelGGL(head_read_vec_kernel<SPV_BF16>, grid, blk, 0, s, p);
    else hipLaunchKernelGGL(head_read_vec_kernel<SPV_F16>, grid, blk, 0, s, p);
    SPV_CHECK_LAUNCH();
    return SPV_OK;
  }
  const size_t work = (size_t)length * num_kv_heads * head_dim, need = (work + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(need < 8192 ? need : 8192)), blk(kThreads);
  if (out_dtype == SPV_F32) hipLaunchKernelGGL(head_read_kernel<SPV_F32>, grid, blk, 0, s, p);
  else if (out_dtype == SPV_BF16) hipLaunchKernelGGL(head_read_kernel<SPV_BF16>, grid, blk, 0, s, p);
  else hipLaunchKernelGGL(head_read_kernel<SPV_F16>, grid, blk, 0, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // extern "C"
