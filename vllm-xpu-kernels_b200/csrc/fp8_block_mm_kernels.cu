// Matrix product of fp8 operands with a scale per block, for NVIDIA B200 (sm_100a), and its C ABI.
//
//   out[m][n] = sum_g  sa[m][g] * sb[n / 128][g] * sum_{k in group g} a[m][k] * b[n][k]        g = 128 columns
//
// a [M, K] are activations with one fp32 scale per row and group (what
// kvc_dynamic_per_token_group_scaled_fp8_quant writes), b [N, K] weights with one per 128 x 128 block.  The scales
// differ from group to group, so a group's products are summed on their own (exactly, or in fp32), multiplied by the
// product of its two scales (one fp32 rounding) and added to an fp32 accumulator (one rounding per group); the result
// is rounded to the output's type once.
#include "kvc_common.cuh"

#include <cuda_fp8.h>

namespace kvc {

constexpr int kMmGroup = 128;  // columns per scale

struct BlockMmParams {
  const unsigned char* a;
  const unsigned char* b;
  const float* a_scales;
  const float* b_scales;
  void* out;
  int64_t m, n, k;
  int64_t a_stride, b_stride, out_stride;  // elements between rows
  int64_t as_stride_m, as_stride_g, bs_stride_n, bs_stride_g;
};

template <int F8>
__device__ __forceinline__ float fp8_to_f32(unsigned char v) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(v, F8 == KVC_KV_FP8_E5M2 ? __NV_E5M2 : __NV_E4M3);
  return __half2float(__half(h));
}

template <typename Tout>
__device__ __forceinline__ Tout from_f32(float v) {
  if constexpr (std::is_same_v<Tout, float>) return v;
  else if constexpr (std::is_same_v<Tout, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

}  // namespace kvc

#include "fp8_block_mm_umma.cuh"

namespace kvc {

// ---------------------------------------------------------------------------------------------
// any shape, stride and alignment: 64 x 64 tiles on the ordinary cores
// ---------------------------------------------------------------------------------------------
constexpr int kPlainTile = 64;
constexpr int kPlainK = 32;

template <int F8, typename Tout>
__global__ void __launch_bounds__(256) block_mm_plain_kernel(const BlockMmParams p) {
  __shared__ float sa[kPlainK][kPlainTile + 4], sb[kPlainK][kPlainTile + 4];
  pdl_prologue();
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kPlainTile, n0 = static_cast<int64_t>(blockIdx.x) * kPlainTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;  // columns 4 tx .., rows 4 ty ..
  float acc[4][4] = {}, part[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kPlainK) {
    __syncthreads();
    for (int i = threadIdx.x; i < kPlainTile * kPlainK; i += 256) {
      const int r = i / kPlainK, c = i % kPlainK;
      sa[c][r] = m0 + r < p.m && k0 + c < p.k ? fp8_to_f32<F8>(__ldg(p.a + (m0 + r) * p.a_stride + k0 + c)) : 0.0f;
      sb[c][r] = n0 + r < p.n && k0 + c < p.k ? fp8_to_f32<F8>(__ldg(p.b + (n0 + r) * p.b_stride + k0 + c)) : 0.0f;
    }
    __syncthreads();
#pragma unroll 8
    for (int c = 0; c < kPlainK; ++c) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = sa[c][4 * ty + i];
        y[i] = sb[c][4 * tx + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = __fmaf_rn(x[i], y[j], part[i][j]);
    }
    if ((k0 + kPlainK) % kMmGroup == 0 || k0 + kPlainK >= p.k) {
      const int64_t g = k0 / kMmGroup;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
          if (m < p.m && n < p.n) {
            const float s = __fmul_rn(__ldg(p.a_scales + m * p.as_stride_m + g * p.as_stride_g),
                                      __ldg(p.b_scales + n / kMmGroup * p.bs_stride_n + g * p.bs_stride_g));
            acc[i][j] = __fmaf_rn(s, part[i][j], acc[i][j]);
          }
          part[i][j] = 0.0f;
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
      if (m < p.m && n < p.n) static_cast<Tout*>(p.out)[m * p.out_stride + n] = from_f32<Tout>(acc[i][j]);
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
namespace {

int mm_fail(const char* text) { return fail(KVC_ERR_INVALID_ARG, std::string("fp8_block_scaled_mm: ") + text); }

template <int F8, typename Tout>
cudaError_t launch_plain(const BlockMmParams& p, cudaStream_t st) {
  BlockMmParams q = p;
  // grid.y is at most 65535: tall products go out in pieces
  const int64_t step = 65535ll * kPlainTile;
  for (int64_t m0 = 0; m0 < p.m; m0 += step) {
    q.m = p.m - m0 < step ? p.m - m0 : step;
    q.a = p.a + m0 * p.a_stride;
    q.a_scales = p.a_scales + m0 * p.as_stride_m;
    q.out = static_cast<Tout*>(p.out) + m0 * p.out_stride;
    const dim3 grid(static_cast<unsigned>((p.n + kPlainTile - 1) / kPlainTile),
                    static_cast<unsigned>((q.m + kPlainTile - 1) / kPlainTile));
    const cudaError_t e = launch_pdl(block_mm_plain_kernel<F8, Tout>, grid, 256, q, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// [rows, k] bytes, rows `stride` apart, boxes of 128 bytes x box_rows.
bool make_mm_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(rows > 1 ? stride : 16)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem_strides[2] = {1, 1};
  return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
                              elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tensor-core kernels need operands that TMA can address.
bool mm_uses_tensor_cores(const BlockMmParams& p) {
  auto rows_ok = [](const void* base, int64_t rows, int64_t stride) {
    return aligned(base, 16) && (rows == 1 || (stride % 16 == 0 && stride > 0 && stride < (1ll << 40)));
  };
  return p.k > 0 && rows_ok(p.a, p.m, p.a_stride) && rows_ok(p.b, p.n, p.b_stride) && tensor_map_encoder() != nullptr;
}

template <typename Params>
cudaError_t launch_umma(void (*kernel)(const BlockMmMaps, const Params), dim3 grid, int threads, int smem, int cluster,
                        const BlockMmMaps& maps, const Params& q, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, q);
}

constexpr int kSms = 148;

// CTAs that a B200 runs at once in clusters of 1 to 8, at one and at two CTAs per SM: what the occupancy calculator says
// of kernels of the same shape.  (Asked about a kernel that allocates tensor memory it always answers one CTA per SM,
// but two do run: 180 CTAs of the 64-token kernel take 40 us where 148 take 36.)
constexpr int kResidentCtas[2][kMaxSplits] = {{148, 148, 135, 132, 130, 132, 105, 120}, {296, 296, 279, 284, 280, 270, 259, 264}};

// What a launch of each tensor-core kernel costs, in hundredths of a microsecond: waves x (a CTA's fixed part + its groups x
// the time of a group).  The constants are fits to times measured on a B200 at sizes from 1 x 2048 x 2048 to 2048 x 10240
// x 8192; they only have to rank the candidates.  The fixed part grows when the accumulators of a cluster are joined, and
// a group takes longer when two CTAs share an SM.
struct MmCost {
  int64_t fixed, joined, group, group_shared;
};
template <int TOK>
constexpr MmCost kThinCost = TOK == 16   ? MmCost{290, 80, 15, 15}
                             : TOK == 32 ? MmCost{360, 80, 20, 20}
                             : TOK == 64 ? MmCost{470, 150, 39, 60}
                                         : MmCost{360, 130, 32, 32};

struct MmPlan {
  int64_t cost = -1;
  int tokens = 0;  // 0: the wide kernel
  int splits = 1;
};

template <int TOK>
void consider_thin(const BlockMmParams& p, MmPlan& best) {
  const int64_t groups = (p.k + kMmGroup - 1) / kMmGroup;
  const int64_t tiles = ((p.n + 127) / 128) * ((p.m + TOK - 1) / TOK);
  if ((p.m + TOK - 1) / TOK > 65535) return;
  for (int s = 1; s <= kMaxSplits && s <= groups; ++s) {
    const int64_t slots = kResidentCtas[ThinCfg<TOK>::kCtasPerSm - 1][s - 1];
    const int64_t waves = (tiles * s + slots - 1) / slots;
    constexpr MmCost c = kThinCost<TOK>;
    const int64_t cost = waves * (c.fixed + (s > 1 ? c.joined : 0) + (groups + s - 1) / s * (tiles * s > kSms ? c.group_shared : c.group));
    if (best.cost < 0 || cost < best.cost) best = MmPlan{cost, TOK, s};
  }
}

MmPlan plan_mm(const BlockMmParams& p) {
  MmPlan best;
  const int64_t groups = (p.k + kMmGroup - 1) / kMmGroup;
  const int64_t wide_tiles = ((p.m + 255) / 256) * ((p.n + 255) / 256);
  if (wide_tiles < (1ll << 30)) best.cost = (wide_tiles + kSms / 2 - 1) / (kSms / 2) * (400 + 47 * groups);
  // a token tile at most twice as large as it has to be, or as small as a quarter of the rows
  if (p.m <= 64) consider_thin<16>(p, best);
  if (p.m > 16 && p.m <= 128) consider_thin<32>(p, best);
  if (p.m > 32) consider_thin<64>(p, best);
  if (p.m > 64) consider_thin<128>(p, best);
  return best;
}

// The CTAs of a cluster that have groups to work on, of `splits` that may have.
int64_t used_splits(int64_t groups, int64_t splits) {
  const int64_t each = (groups + splits - 1) / splits;
  return (groups + each - 1) / each;
}

template <int F8, typename Tout, int TOK>
cudaError_t launch_thin(const BlockMmParams& p, int64_t splits, bool& encoded, cudaStream_t st) {
  BlockMmMaps maps;
  encoded = make_mm_map(&maps.a, p.a, p.m, p.k, p.a_stride, TOK) && make_mm_map(&maps.b, p.b, p.n, p.k, p.b_stride, 128);
  if (!encoded) return cudaSuccess;
  const int64_t groups = (p.k + kMmGroup - 1) / kMmGroup;
  const int64_t n_tiles = (p.n + 127) / 128, m_tiles = (p.m + TOK - 1) / TOK;
  ThinParams q{};
  q.a_scales = p.a_scales;
  q.b_scales = p.b_scales;
  q.out = p.out;
  q.out_stride = p.out_stride;
  q.as_stride_m = p.as_stride_m;
  q.as_stride_g = p.as_stride_g;
  q.bs_stride_n = p.bs_stride_n;
  q.bs_stride_g = p.bs_stride_g;
  q.m = static_cast<int32_t>(p.m);
  q.n = static_cast<int32_t>(p.n);
  q.groups = static_cast<int32_t>(groups);
  q.groups_per_split = static_cast<int32_t>((groups + splits - 1) / splits);
  q.splits = static_cast<int32_t>(used_splits(groups, splits));
  q.own = (TOK + q.splits - 1) / q.splits;
  q.wide_stores = aligned(p.out, 16) && (p.out_stride * (int64_t)sizeof(Tout)) % 16 == 0;
  return launch_umma(block_mm_thin_kernel<F8, Tout, TOK>, dim3(static_cast<unsigned>(n_tiles * q.splits), static_cast<unsigned>(m_tiles)),
                     ThinCfg<TOK>::kThreads, ThinCfg<TOK>::kSmem, q.splits, maps, q, st);
}

template <int F8, typename Tout>
cudaError_t launch_wide(const BlockMmParams& p, bool& encoded, cudaStream_t st) {
  BlockMmMaps maps;
  encoded = make_mm_map(&maps.a, p.a, p.m, p.k, p.a_stride, 128) && make_mm_map(&maps.b, p.b, p.n, p.k, p.b_stride, 128);
  if (!encoded) return cudaSuccess;
  WideParams q{};
  q.a_scales = p.a_scales;
  q.b_scales = p.b_scales;
  q.out = p.out;
  q.out_stride = p.out_stride;
  q.as_stride_m = p.as_stride_m;
  q.as_stride_g = p.as_stride_g;
  q.bs_stride_n = p.bs_stride_n;
  q.bs_stride_g = p.bs_stride_g;
  q.m = static_cast<int32_t>(p.m);
  q.n = static_cast<int32_t>(p.n);
  q.groups = static_cast<int32_t>((p.k + kMmGroup - 1) / kMmGroup);
  q.m_tiles = static_cast<int32_t>((p.m + 255) / 256);
  q.n_tiles = static_cast<int32_t>((p.n + 255) / 256);
  q.store_bytes = 32;
  while (q.store_bytes > 8 && !(aligned(p.out, q.store_bytes) && (p.out_stride * (int64_t)sizeof(Tout)) % q.store_bytes == 0))
    q.store_bytes /= 2;
  const int64_t tiles = static_cast<int64_t>(q.m_tiles) * q.n_tiles;
  const int64_t pairs = tiles < kSms / 2 ? tiles : kSms / 2;
  return launch_umma(block_mm_wide_kernel<F8, Tout>, dim3(static_cast<unsigned>(2 * pairs)), kWideThreads, WideCfg::kSmem, 2,
                     maps, q, st);
}

template <int F8, typename Tout>
cudaError_t launch_mm(const BlockMmParams& p, cudaStream_t st) {
  if (mm_uses_tensor_cores(p)) {
    bool encoded = false;
    cudaError_t e;
    const MmPlan plan = plan_mm(p);
    switch (plan.tokens) {
      case 16: e = launch_thin<F8, Tout, 16>(p, plan.splits, encoded, st); break;
      case 32: e = launch_thin<F8, Tout, 32>(p, plan.splits, encoded, st); break;
      case 64: e = launch_thin<F8, Tout, 64>(p, plan.splits, encoded, st); break;
      case 128: e = launch_thin<F8, Tout, 128>(p, plan.splits, encoded, st); break;
      default: e = plan.cost >= 0 ? launch_wide<F8, Tout>(p, encoded, st) : cudaSuccess; break;
    }
    if (encoded) return e;
  }
  return launch_plain<F8, Tout>(p, st);
}

template <int F8>
cudaError_t launch_mm_out(int out_dtype, const BlockMmParams& p, cudaStream_t st) {
  if (out_dtype == KVC_IN_F32) return launch_mm<F8, float>(p, st);
  if (out_dtype == KVC_IN_F16) return launch_mm<F8, __half>(p, st);
  return launch_mm<F8, __nv_bfloat16>(p, st);
}

}  // namespace
}  // namespace kvc

extern "C" {

KVC_API int kvc_fp8_block_scaled_mm_device_status(int* status) {
  if (!status) return kvc::mm_fail("status must be non-NULL");
  int v = 0;
  cudaError_t e = cudaDeviceSynchronize();  // non-blocking streams too, which the copy alone would not wait for
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, kvc::g_block_mm_status, sizeof(int));
  if (e != cudaSuccess)
    return kvc::fail(KVC_ERR_CUDA, std::string("fp8_block_scaled_mm_device_status: ") + cudaGetErrorString(e));
  *status = v;
  return KVC_OK;
}

KVC_API int kvc_fp8_block_scaled_mm_clear_device_status(void) {
  const int zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(kvc::g_block_mm_status, &zero, sizeof(int));
  if (e != cudaSuccess)
    return kvc::fail(KVC_ERR_CUDA, std::string("fp8_block_scaled_mm_clear_device_status: ") + cudaGetErrorString(e));
  return KVC_OK;
}

KVC_API int kvc_fp8_block_scaled_mm_plan(int64_t m, int64_t n, int64_t k, int32_t* tile_tokens, int32_t* splits) {
  using namespace kvc;
  if (m < 1 || n < 1 || k < 1 || m > 0x3FFFFFFFll || n > 0x3FFFFFFFll || k > 0x3FFFFFFFll)
    return fail(KVC_ERR_INVALID_ARG, "fp8_block_scaled_mm_plan: sizes out of range");
  BlockMmParams p{};
  p.m = m;
  p.n = n;
  p.k = k;
  const MmPlan plan = plan_mm(p);
  const int64_t groups = (k + kMmGroup - 1) / kMmGroup;
  if (tile_tokens) *tile_tokens = plan.tokens > 0 ? plan.tokens : 256;
  if (splits) *splits = static_cast<int32_t>(plan.tokens > 0 ? used_splits(groups, plan.splits) : 1);
  return KVC_OK;
}

KVC_API int kvc_fp8_block_scaled_mm_selftest_gives_up(int64_t tries, void* stream) {
  if (tries < 1 || tries > 5000)
    return kvc::fail(KVC_ERR_INVALID_ARG,
                     "fp8_block_scaled_mm_selftest_gives_up: tries must be within 1..5000 (about 20 us each)");
  kvc::block_mm_gives_up_kernel<<<1, 128, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<uint32_t>(tries));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return kvc::fail(KVC_ERR_CUDA,
                     std::string("fp8_block_scaled_mm_selftest_gives_up launch failed: ") + cudaGetErrorString(e));
  return KVC_OK;
}

KVC_API int kvc_fp8_block_scaled_mm(void* out, const void* a, const void* b, const float* a_scales,
                                    const float* b_scales, int64_t m, int64_t n, int64_t k, int64_t out_stride,
                                    int64_t a_stride, int64_t b_stride, int64_t a_scale_stride_m,
                                    int64_t a_scale_stride_g, int64_t b_scale_stride_n, int64_t b_scale_stride_g,
                                    int out_dtype, int fp8_dtype, void* stream) {
  using namespace kvc;
  if (out_dtype != KVC_IN_F32 && out_dtype != KVC_IN_F16 && out_dtype != KVC_IN_BF16)
    return fail(KVC_ERR_UNSUPPORTED, "fp8_block_scaled_mm: unsupported output type code " + std::to_string(out_dtype));
  if (fp8_dtype != KVC_KV_FP8_E4M3 && fp8_dtype != KVC_KV_FP8_E5M2)
    return fail(KVC_ERR_UNSUPPORTED, "fp8_block_scaled_mm: the operands must be fp8_e4m3 or fp8_e5m2");
  if (m < 0 || n < 0 || k < 0) return mm_fail("negative size");
  if (m > 0x3FFFFFFFll || n > 0x3FFFFFFFll || k > 0x3FFFFFFFll) return mm_fail("sizes out of range");
  if (m == 0 || n == 0) return KVC_OK;
  if (!out || (k > 0 && (!a || !b || !a_scales || !b_scales))) return mm_fail("out, a, b and the scales must be non-NULL");
  if (!aligned(out, in_elem_size(out_dtype)) || !aligned(a_scales, 4) || !aligned(b_scales, 4))
    return mm_fail("out and the scales must be aligned to their element size");
  BlockMmParams p{};
  p.a = static_cast<const unsigned char*>(a);
  p.b = static_cast<const unsigned char*>(b);
  p.a_scales = a_scales;
  p.b_scales = b_scales;
  p.out = out;
  p.m = m;
  p.n = n;
  p.k = k;
  p.a_stride = a_stride;
  p.b_stride = b_stride;
  p.out_stride = out_stride;
  p.as_stride_m = a_scale_stride_m;
  p.as_stride_g = a_scale_stride_g;
  p.bs_stride_n = b_scale_stride_n;
  p.bs_stride_g = b_scale_stride_g;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = fp8_dtype == KVC_KV_FP8_E5M2 ? launch_mm_out<KVC_KV_FP8_E5M2>(out_dtype, p, st)
                                                     : launch_mm_out<KVC_KV_FP8_E4M3>(out_dtype, p, st);
  if (e != cudaSuccess) return fail(KVC_ERR_CUDA, std::string("fp8_block_scaled_mm launch failed: ") + cudaGetErrorString(e));
  return KVC_OK;
}

}  // extern "C"
