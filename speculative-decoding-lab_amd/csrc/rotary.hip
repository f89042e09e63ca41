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
// turns. What is left of a turn goes to fp32 sin and cos (an error of 2^-24
// turns at most), the products are fp32, and each result is rounded once.
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

// cos and sin of position * inv_freq_i, times the factor.
__device__ __forceinline__ float2 turn_of(const RotaryParams& p, int b, int j, int i) {
  const int axis = p.axis_of ? min(max(p.axis_of[i], 0), p.axes - 1) : 0;
  const int pos = p.positions ? p.positions[((size_t)axis * p.B + b) * p.C + j] : p.start[b] + j;
  const double t = (double)pos * (p.inv_freq[i] * kInvTwoPi);
  const float f = (float)(t - __builtin_rint(t));  // turns, in [-1/2, 1/2]
  float s, c;
  sincospif(2.f * f, &s, &c);
  return make_float2(c * p.factor, s * p.factor);
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
      put(e0, a * t.x - c * t.y);
      put(e1, c * t.x + a * t.y);
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
