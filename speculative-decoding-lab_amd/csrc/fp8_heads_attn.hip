// Causal attention of a chunk over an 8-bit paged cache with a scale for each
// (block, head).
//
// Row (j, r) of kv head h (query head h * ratio + r, chunk token j) attends keys
// 0 .. start + j:  z_i = scale * s_k(i) * (q . k_i),  p = softmax(z),
// o = sum_i p_i s_v(i) v_i,  with k_i, v_i the decoded codes and s_k, s_v the
// scales of key i's block. Scores, the running maximum and sum and the output are
// held in fp32.
#include "fp8_heads.h"

using namespace spv;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct HeadAttn {
  void* out;
  const void* q;
  const uint8_t* kpool;
  const uint8_t* vpool;
  const float* scales;
  const int32_t* tables;
  const int32_t* seq_ids;
  const int32_t* start;
  const int32_t* lens;
  int32_t* ctr;
  int maxb, B, C, Hq, Hkv, ratio, d, bs, layer, cap, max_ctx;
  float scale_log2;
};

// A read the contract forbids is recorded as 1 + the entry's index; such a page
// reads block 0 instead.
__device__ __forceinline__ void flag_read(const HeadAttn& p, int b) {
  if (p.ctr) p.ctr[CTR_BAD_READ] = b + 1;
}
__device__ __forceinline__ int block_of(const HeadAttn& p, int sid, int blk, int b) {
  const int id = p.tables[(size_t)sid * p.maxb + min(blk, p.maxb - 1)];
  if ((unsigned)id < (unsigned)p.cap) return id;
  flag_read(p, b);
  return 0;
}

// One wave per row, 64 keys at a time, any head_dim, block size and ratio.
constexpr int kAnyRows = 4;
template <int QT>
__global__ __launch_bounds__(64 * kAnyRows) void head_attn_any_kernel(HeadAttn p, int groups) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ float s_w[kAnyRows][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = p.d;
  const int g = blockIdx.x % groups, bh = blockIdx.x / groups, h = bh % p.Hkv, b = bh / p.Hkv;
  const int row = g * kAnyRows + wave, start = p.start[b], sid = p.seq_ids[b];
  if (g == 0 && h == 0 && threadIdx.x == 0 &&
      (start < 0 || start + p.C > p.max_ctx || (p.lens && start + p.C > p.lens[sid])))
    flag_read(p, b);
  if (row >= p.C * p.ratio) return;  // whole waves; no barrier below
  const int j = row / p.ratio, hq = h * p.ratio + row - j * p.ratio;
  float* const q = reinterpret_cast<float*>(lds) + (size_t)wave * 2 * d;
  float* const o = q + d;
  const size_t at = (((size_t)b * p.C + j) * p.Hq + hq) * d;
  for (int e = lane; e < d; e += 64) {
    q[e] = load_elem<QT>(p.q, at + e) * p.scale_log2;
    o[e] = 0.f;
  }
  const int n = min(start + j + 1, p.max_ctx);
  float m = -INFINITY, l = 0.f;
  for (int base = 0; base < n; base += 64) {
    const int key = base + lane;
    float z = -INFINITY, vs = 0.f;
    if (key < n) {
      const int blk = key / p.bs, off = key - blk * p.bs, phys = block_of(p, sid, blk, b);
      const float* const s = p.scales + scale_of(p.layer, p.cap, phys, p.Hkv, h);
      const uint8_t* const k = p.kpool + page_of(p.layer, p.cap, phys, p.Hkv, h, p.bs, d) + (size_t)off * d;
      float dot = 0.f;
      for (int e = 0; e < d; ++e) dot = fmaf(q[e], fp8e4m3_to_f32(k[e]), dot);
      z = dot * s[0];
      vs = s[1];
    }
    float top = z;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    const float w = exp2f(z - ref), keep = exp2f(m - ref);
    float sum = w;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    l = l * keep + sum;
    m = mn;
    s_w[wave][lane] = w * vs;
    __builtin_amdgcn_wave_barrier();
    for (int e = lane; e < d; e += 64) {
      float acc = o[e] * keep;
      for (int i = 0; i < min(64, n - base); ++i) {
        const int blk = (base + i) / p.bs, off = base + i - blk * p.bs, phys = block_of(p, sid, blk, b);
        const uint8_t* const v = p.vpool + page_of(p.layer, p.cap, phys, p.Hkv, h, p.bs, d);
        acc = fmaf(s_w[wave][i], fp8e4m3_to_f32(v[(size_t)e * p.bs + off]), acc);
      }
      o[e] = acc;
    }
    __builtin_amdgcn_wave_barrier();
  }
  const float inv = n > 0 ? 1.f / l : 0.f;
  for (int e = lane; e < d; e += 64) store_elem<QT>(p.out, at + e, o[e] * inv);
}

}  // namespace

extern "C" {

size_t spv_verify_attn_fp8_heads_workspace_bytes(int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
                                                 int32_t head_dim, int32_t block_size, int32_t max_ctx) {
  (void)B, (void)C, (void)num_q_heads, (void)num_kv_heads, (void)head_dim, (void)block_size, (void)max_ctx;
  return 0;
}

int spv_verify_attn_fp8_heads(void* out, const void* q, int q_dtype, const void* k_pool, const void* v_pool,
                              const float* kv_scales, const int32_t* block_tables, int32_t max_blocks_per_seq,
                              const int32_t* seq_ids, const int32_t* start_pos, const int32_t* seq_lens, int32_t* ctr,
                              int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, int32_t layer, int32_t capacity, int32_t max_ctx, float scale,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (!out || !q || !k_pool || !v_pool || !kv_scales || !block_tables || !seq_ids || !start_pos || B < 0 || C < 1 ||
      num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads || head_dim < 1 || block_size < 1 ||
      layer < 0 || capacity < 1 || max_blocks_per_seq < 1 || max_ctx < 1)
    return SPV_ERR_ARG;
  if (q_dtype != SPV_F32 && q_dtype != SPV_BF16 && q_dtype != SPV_F16) return SPV_ERR_ARG;
  if ((max_ctx + (long long)block_size - 1) / block_size > max_blocks_per_seq) return SPV_ERR_ARG;
  if (head_dim > 2048) return SPV_ERR_UNSUPPORTED;
  const int ratio = num_q_heads / num_kv_heads;
  const long long groups = ((long long)C * ratio + kAnyRows - 1) / kAnyRows, grid = groups * num_kv_heads * B;
  if ((long long)C * ratio > 0x3fffffffLL || grid > 0x7fffffffLL) return SPV_ERR_ARG;
  if (B == 0) return SPV_OK;
  (void)workspace, (void)workspace_bytes;
  const HeadAttn p{out, q, static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), kv_scales,
                   block_tables, seq_ids, start_pos, seq_lens, ctr, max_blocks_per_seq, B, C, num_q_heads,
                   num_kv_heads, ratio, head_dim, block_size, layer, capacity, max_ctx, scale * kLog2e};
  const size_t smem = (size_t)kAnyRows * 2 * head_dim * sizeof(float);
  hipStream_t s = (hipStream_t)stream;
#define SPV_ANY(QT) \
  hipLaunchKernelGGL(head_attn_any_kernel<QT>, dim3((unsigned)grid), dim3(64 * kAnyRows), smem, s, p, (int)groups)
  if (q_dtype == SPV_F32) SPV_ANY(SPV_F32);
  else if (q_dtype == SPV_BF16) SPV_ANY(SPV_BF16);
  else SPV_ANY(SPV_F16);
#undef SPV_ANY
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // extern "C"
