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
// With head norms (NORM) the row turned is y_e = x_e w_e / sqrt(mean x^2 + eps),
// w the query heads' or the key heads' weights: the sum of squares, the factor
// and the products are fp32, and nothing is rounded between the norm and the turn.
//
// The angle is formed and reduced in fp64: at position 10^6 the fp32 product is
// off by up to 0.03 rad, and the fp64 one, in turns, by 2^-53 of some 10^5
// turns. What is left of a turn, in fp32, goes to fp32 sin and cos, and what that rounding
// leaves (up to 2^-26 turns, as much as the rounding of sin and cos) to their first-order terms;
// the products are fp32, and each result is rounded once.
#include "rotary_common.h"

using namespace spv;

namespace {

// One thread per element pair (or element past the rotary width) of a row; one
// workgroup per (entry, token), with NORM one wave per row. Any head_dim, stride
// and alignment.
template <int DT, int KO, bool APPEND, bool NORM>
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
  // Item i of the row of head hh (the query heads first): a pair, or an element past the width.
  struct Row {
    const uint8_t* src;
    size_t in, out;
    bool isq;
  };
  auto row_of = [&](int hh, Row& w) {  // false: nothing to do for this head
    w.isq = hh < p.Hq;
    const int h = w.isq ? hh : hh - p.Hq;
    w.src = w.isq ? p.q : p.k;
    if (!w.src || (APPEND && !w.isq && row < 0)) return false;
    const long long* st = w.isq ? p.qs : p.ks;
    w.in = (size_t)((long long)b * st[0] + (long long)j * st[1] + (long long)h * st[2]);
    if (w.isq) w.out = (size_t)((long long)b * p.qos[0] + (long long)j * p.qos[1] + (long long)h * p.qos[2]);
    else if constexpr (APPEND) w.out = ((((size_t)p.layer * p.cap + blk) * p.Hkv + h) * p.bs + off) * p.d;
    else w.out = (size_t)((long long)b * p.kos[0] + (long long)j * p.kos[1] + (long long)h * p.kos[2]);
    return true;
  };
  auto do_item = [&](const Row& w, int i, float inv) {
    auto get = [&](int e) {
      const float x = load_elem<DT>(w.src, w.in + e);
      if constexpr (!NORM) return x;
      const float* const wt = w.isq ? p.wq : p.wk;
      return x * (wt ? inv * wt[e] : inv);
    };
    auto put = [&](int e, float x) {
      if (w.isq) store_elem<DT>(p.q_out, w.out + e, x);
      else if constexpr (APPEND) store_elem<DT>(p.kpool, w.out + e, x);
      else store_elem<KO>(p.k_out, w.out + e, x);
    };
    if (i < half) {
      const int e0 = p.interleaved ? 2 * i : i, e1 = p.interleaved ? 2 * i + 1 : i + half;
      const float a = get(e0), c = get(e1);
      const float2 t = turn_of(p, b, j, i);
      const float2 y = turned(a, c, t);
      put(e0, y.x);
      put(e1, y.y);
    } else {
      const int e = p.R + (i - half);
      put(e, get(e));
    }
  };
  Row w;
  if constexpr (NORM) {
    const int lane = threadIdx.x & 63;
    for (int hh = threadIdx.x >> 6; hh < p.Hq + p.Hkv; hh += blockDim.x >> 6) {
      if (!row_of(hh, w)) continue;
      float ss = 0.f;
      for (int e = lane; e < p.d; e += 64) {
        const float x = load_elem<DT>(w.src, w.in + e);
        ss = fmaf(x, x, ss);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
      const float inv = norm_factor(ss, p.d, p.eps);
      for (int i = lane; i < items; i += 64) do_item(w, i, inv);
    }
  } else {
    for (int it = threadIdx.x; it < (p.Hq + p.Hkv) * items; it += blockDim.x) {
      const int hh = it / items;
      if (row_of(hh, w)) do_item(w, it - hh * items, 1.f);
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

template <int DT, bool APPEND, bool NORM>
__global__ __launch_bounds__(kVecThreads) void rotary_vec_kernel(RotaryParams p, VecShape v) {
  extern __shared__ __align__(16) uint8_t lds[];
  rotary_vec_rows<DT, APPEND, NORM>(p, v, blockIdx.x, blockIdx.y, lds);
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

template <bool APPEND, bool NORM>
void launch_vec(const RotaryParams& p, const VecShape& v, int dtype, hipStream_t s) {
  const size_t smem = vec_lds(p, v, dtype_size(dtype), APPEND, NORM);
  const dim3 grid((unsigned)(p.B * v.tiles), (unsigned)(v.slices + (APPEND ? p.Hkv : 0))), blk(kVecThreads);
#define SPV_VEC(DT) hipLaunchKernelGGL((rotary_vec_kernel<DT, APPEND, NORM>), grid, blk, smem, s, p, v)
  if (dtype == SPV_F32) SPV_VEC(SPV_F32);
  else if (dtype == SPV_BF16) SPV_VEC(SPV_BF16);
  else SPV_VEC(SPV_F16);
#undef SPV_VEC
}

template <bool NORM>
void launch_dense(const RotaryParams& p, int dtype, int k_out_dtype, hipStream_t s) {
  VecShape v;
  if (k_out_dtype == dtype && vec_shape(p, dtype_size(dtype), false, NORM, v)) {
    launch_vec<false, NORM>(p, v, dtype, s);
    return;
  }
  const dim3 grid((unsigned)(p.B * p.C)), blk(256);
#define SPV_ROT(DT, KO) hipLaunchKernelGGL((rotary_elem_kernel<DT, KO, false, NORM>), grid, blk, 0, s, p)
  if (dtype == SPV_F32) SPV_ROT(SPV_F32, SPV_F32);
  else if (dtype == SPV_BF16 && k_out_dtype == SPV_BF16) SPV_ROT(SPV_BF16, SPV_BF16);
  else if (dtype == SPV_BF16) SPV_ROT(SPV_BF16, SPV_F32);
  else if (k_out_dtype == SPV_F16) SPV_ROT(SPV_F16, SPV_F16);
  else SPV_ROT(SPV_F16, SPV_F32);
#undef SPV_ROT
}

template <bool NORM>
void launch_append(const RotaryParams& p, int dtype, hipStream_t s) {
  VecShape v;
  if (vec_shape(p, dtype_size(dtype), true, NORM, v)) {
    launch_vec<true, NORM>(p, v, dtype, s);
    return;
  }
  const dim3 grid((unsigned)(p.B * p.C)), blk(256);
#define SPV_ROT(DT) hipLaunchKernelGGL((rotary_elem_kernel<DT, DT, true, NORM>), grid, blk, 0, s, p)
  if (dtype == SPV_F32) SPV_ROT(SPV_F32);
  else if (dtype == SPV_BF16) SPV_ROT(SPV_BF16);
  else SPV_ROT(SPV_F16);
#undef SPV_ROT
}

// The norm's part of a call; NULL where the rows are only rotated.
struct NormArgs {
  const float* wq;
  const float* wk;
  float eps;
};

bool norm_ok(const NormArgs* n) { return !n || (n->eps >= 0.f && n->eps < 1e30f); }

void set_norm(RotaryParams& p, const NormArgs* n) {
  if (!n) return;
  p.wq = n->wq;
  p.wk = n->wk;
  p.eps = n->eps;
}

void set_strides(long long* dst, const int64_t* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}

int rotary_impl(const NormArgs* norm, void* q_out, const void* q, void* k_out, const void* k, int dtype, int k_out_dtype,
               const int64_t* strides, const int32_t* positions, const double* inv_freq, const int32_t* axis_of,
               int32_t axes, float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
               int32_t head_dim, int32_t rotary_dim, int32_t interleaved, void* stream) {
  if (!strides || !positions || (!q && !k) || (q && !q_out) || (k && !k_out) || !norm_ok(norm)) return SPV_ERR_ARG;
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
  set_norm(p, norm);
  hipStream_t s = (hipStream_t)stream;
  if (norm) launch_dense<true>(p, dtype, k_out_dtype, s);
  else launch_dense<false>(p, dtype, k_out_dtype, s);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

int rotary_append_impl(const NormArgs* norm, void* q_out, const void* q, const void* k_new, const void* v_new, int dtype,
                         const int64_t* strides, void* k_pool, void* v_pool, int32_t* block_tables,
                         int32_t max_blocks_per_seq, int32_t* num_blocks, int32_t* seq_lens, int32_t* free_stack,
                         int32_t* free_flag, int32_t* ctr, const int32_t* seq_ids, const int32_t* start_pos,
                         const int32_t* positions, const double* inv_freq, const int32_t* axis_of, int32_t axes,
                         float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
                         int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int32_t layer, int32_t capacity,
                         int32_t block_size, int32_t may_alloc, int32_t follow_plan, int32_t* write_plan,
                         void* stream) {
  if (!strides || !k_new || !v_new || (q && !q_out) || !k_pool || !v_pool || !block_tables || !num_blocks ||
      !seq_lens || !ctr || !seq_ids || !start_pos || (follow_plan && (!write_plan || may_alloc)) || !norm_ok(norm))
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
  set_norm(p, norm);
  hipStream_t s = (hipStream_t)stream;
  if (norm) launch_append<true>(p, dtype, s);
  else launch_append<false>(p, dtype, s);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // namespace

namespace spv {

int rotary_queries(const RotaryParams& p, int dtype, bool norm, hipStream_t s) {
  if (norm) launch_dense<true>(p, dtype, dtype, s);
  else launch_dense<false>(p, dtype, dtype, s);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // namespace spv

extern "C" {

int spv_rotary(void* q_out, const void* q, void* k_out, const void* k, int dtype, int k_out_dtype,
               const int64_t* strides, const int32_t* positions, const double* inv_freq, const int32_t* axis_of,
               int32_t axes, float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
               int32_t head_dim, int32_t rotary_dim, int32_t interleaved, void* stream) {
  return rotary_impl(nullptr, q_out, q, k_out, k, dtype, k_out_dtype, strides, positions, inv_freq, axis_of, axes,
                     factor, B, C, num_q_heads, num_kv_heads, head_dim, rotary_dim, interleaved, stream);
}

int spv_norm_rotary(void* q_out, const void* q, void* k_out, const void* k, int dtype, int k_out_dtype,
                    const int64_t* strides, const float* q_weight, const float* k_weight, float eps,
                    const int32_t* positions, const double* inv_freq, const int32_t* axis_of, int32_t axes,
                    float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                    int32_t rotary_dim, int32_t interleaved, void* stream) {
  const NormArgs norm{q_weight, k_weight, eps};
  return rotary_impl(&norm, q_out, q, k_out, k, dtype, k_out_dtype, strides, positions, inv_freq, axis_of, axes,
                     factor, B, C, num_q_heads, num_kv_heads, head_dim, rotary_dim, interleaved, stream);
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
  return rotary_append_impl(nullptr, q_out, q, k_new, v_new, dtype, strides, k_pool, v_pool, block_tables,
                            max_blocks_per_seq, num_blocks, seq_lens, free_stack, free_flag, ctr, seq_ids, start_pos,
                            positions, inv_freq, axis_of, axes, factor, B, C, num_q_heads, num_kv_heads, head_dim,
                            rotary_dim, interleaved, layer, capacity, block_size, may_alloc, follow_plan, write_plan,
                            stream);
}

int spv_kv_norm_rotary_append(void* q_out, const void* q, const void* k_new, const void* v_new, int dtype,
                              const int64_t* strides, const float* q_weight, const float* k_weight, float eps,
                              void* k_pool, void* v_pool, int32_t* block_tables, int32_t max_blocks_per_seq,
                              int32_t* num_blocks, int32_t* seq_lens, int32_t* free_stack, int32_t* free_flag,
                              int32_t* ctr, const int32_t* seq_ids, const int32_t* start_pos,
                              const int32_t* positions, const double* inv_freq, const int32_t* axis_of, int32_t axes,
                              float factor, int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
                              int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int32_t layer,
                              int32_t capacity, int32_t block_size, int32_t may_alloc, int32_t follow_plan,
                              int32_t* write_plan, void* stream) {
  const NormArgs norm{q_weight, k_weight, eps};
  return rotary_append_impl(&norm, q_out, q, k_new, v_new, dtype, strides, k_pool, v_pool, block_tables,
                            max_blocks_per_seq, num_blocks, seq_lens, free_stack, free_flag, ctr, seq_ids, start_pos,
                            positions, inv_freq, axis_of, axes, factor, B, C, num_q_heads, num_kv_heads, head_dim,
                            rotary_dim, interleaved, layer, capacity, block_size, may_alloc, follow_plan, write_plan,
                            stream);
}

}  // extern "C"
