// Rotary position embedding with several position axes (time, height, width of images and video) for NVIDIA B200
// (sm_100a), alone and fused with the paged KV-cache write, and their C ABI.
//
//   kvc_multi_axis_rotary_embedding                  query [T, Hq, D] and key [T, Hkv, D], in place or to other tensors
//   kvc_multi_axis_rotary_embedding_and_cache_flash  the same, and the rotated key and the value go to their cache
//                                                    slots (flash layout) in the same pass
//
// A token has one position per axis, and every frequency i < rot_dim / 2 belongs to one axis:
//   x' = x*c - y*s   y' = y*c + x*s   with c, s = cos_sin_cache[positions[axis(i)][t]][i | rot_dim/2 + i]
// Pairs (x, y) are elements (i, i + rot_dim/2) in the GPT-NeoX style and (2i, 2i+1) in the GPT-J style.  The products
// and the sum are fp32 and the result is rounded to the tensors' type ONCE.  (rotary_embedding, whose contract is an
// elementwise tensor expression in the tensors' type, rounds three times; rounding once costs nothing here, the
// kernels wait for memory, and halves the error.)  An axis whose position lies outside the table leaves its
// frequencies unrotated.
//
// Pure HBM traffic: rows are read and written once.  The reference plugin has no counterpart.
#include "kvc_common.cuh"
#include "kvc_convert.cuh"

namespace kvc {

constexpr int kAxesMax = 4;
constexpr int kAxesMaxHalf = 512;  // rot_dim <= 1024
constexpr int kAxesThreads = 128;
constexpr int kAxesItems = 8;  // pieces of heads a thread rotates

struct AxesParams {
  const int64_t* positions;
  const void* query;
  const void* key;
  void* query_out;  // == query when in place
  void* key_out;    // NULL: the rotated key goes to the cache only
  const void* cos_sin_cache;
  const void* value;
  void* key_cache;
  void* value_cache;
  const int64_t* slot_mapping;
  const float* k_scale;
  const float* v_scale;
  int64_t position_stride, max_position, num_slot_tokens;
  int64_t query_stride_t, query_stride_h, key_stride_t, key_stride_h;  // elements
  int64_t qout_stride_t, qout_stride_h, kout_stride_t, kout_stride_h;
  int64_t value_stride_t, value_stride_h;
  int64_t block_stride, page_stride, head_stride, block_size;
  uint32_t axis_of[kAxesMaxHalf / 16];  // two bits per frequency
  int32_t rot_dim, half, bs_shift;
  uint32_t num_q_heads, num_heads;  // query heads; query and key heads
  uint32_t chunks;                  // pieces of a head
  uint32_t rows;                    // tokens * heads of this launch
  uint32_t rows_per_cta;
  // items behind the rotation: elements that are only copied.  Per token: query tails, key tails, value rows
  uint32_t tail_chunks, value_chunks;
  uint32_t seg_key, seg_value, copy_per_token, copy_items;
  uint32_t rot_ctas;
  FastDiv div_chunks, div_heads, div_half, div_copy, div_tail, div_value;
  bool table_f32;
};

template <typename T>
__device__ __forceinline__ void put_float(unsigned char* p, float v) {
  if constexpr (std::is_same_v<T, float>) *reinterpret_cast<float*>(p) = v;
  else if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<__half*>(p) = __float2half_rn(v);
  else *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
}

// two values as one 32-bit word of 16-bit floats, `lo` in bits 0..15; round to nearest even
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t w;
  if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}

template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  float2 f;
  unpack2<T>(w, f.x, f.y);
  return f;
}

// BYTES bytes as one access, or (ALIGNED false) element by element.
template <typename T, bool ALIGNED, int BYTES>
__device__ __forceinline__ void load_elements(Chunk<BYTES>& c, const T* src) {
  if constexpr (ALIGNED) load_chunk_inplace(c, src);
  else {
#pragma unroll
    for (int j = 0; j < BYTES / (int)sizeof(T); ++j) {
      Chunk<(int)sizeof(T)> one;
      load_chunk_inplace(one, src + j);
#pragma unroll
      for (int b = 0; b < (int)sizeof(T); ++b) c.b[j * (int)sizeof(T) + b] = one.b[b];
    }
  }
}
template <bool ALIGNED, int ELEM, int BYTES>
__device__ __forceinline__ void store_elements(char* dst, const Chunk<BYTES>& c) {
  if constexpr (ALIGNED) store_chunk(dst, c, true);
  else {
#pragma unroll
    for (int j = 0; j < BYTES / ELEM; ++j) store_piece<ELEM>(dst + j * ELEM, c, j * ELEM);
  }
}

// The cosines and sines of `count` tokens from `first` on, [token][cosines, then sines], each frequency by the position of
// its axis; off[token] bit a: axis a's position lies outside the table.  One element per thread and step: neighbouring
// threads read neighbouring frequencies, of two or three table rows where the axes are interleaved.
template <typename Tcs>
__device__ __forceinline__ void gather_turns(const AxesParams& p, Tcs* turns, uint32_t* off, uint32_t first, uint32_t count) {
  const Tcs* table = static_cast<const Tcs*>(p.cos_sin_cache);
  for (uint32_t e = threadIdx.x; e < count * p.half; e += kAxesThreads) {
    const uint32_t tok = p.div_half.div(e);
    const uint32_t i = e - tok * p.half;
    const uint32_t axis = (p.axis_of[i >> 4] >> (2 * (i & 15))) & 3u;
    const int64_t pos = __ldg(p.positions + axis * p.position_stride + first + tok);
    if (pos >= 0 && pos < p.max_position) {
      turns[tok * p.rot_dim + i] = table[pos * p.rot_dim + i];
      turns[tok * p.rot_dim + p.half + i] = table[pos * p.rot_dim + p.half + i];
    } else {
      atomicOr(off + tok, 1u << axis);
    }
  }
}

// F cosines and sines of one token; bit j of the result: frequency f0 + j is not rotated.
template <typename Tcs, int F, bool ALIGNED>
__device__ __forceinline__ void read_turns(const Tcs* turns, int half, float (&c)[F], float (&s)[F]) {
  if constexpr (ALIGNED && F * (int)sizeof(Tcs) <= 16 && F > 1) {
    const Chunk<F * (int)sizeof(Tcs)> cv = *reinterpret_cast<const Chunk<F * (int)sizeof(Tcs)>*>(turns);
    const Chunk<F * (int)sizeof(Tcs)> sv = *reinterpret_cast<const Chunk<F * (int)sizeof(Tcs)>*>(turns + half);
#pragma unroll
    for (int j = 0; j < F; ++j) {
      c[j] = to_f32<Tcs>(cv.b + j * (int)sizeof(Tcs));
      s[j] = to_f32<Tcs>(sv.b + j * (int)sizeof(Tcs));
    }
  } else {
#pragma unroll
    for (int j = 0; j < F; ++j) {
      c[j] = to_f32<Tcs>(reinterpret_cast<const unsigned char*>(turns + j));
      s[j] = to_f32<Tcs>(reinterpret_cast<const unsigned char*>(turns + half + j));
    }
  }
}
template <int F>
__device__ __forceinline__ uint32_t still_mask(const AxesParams& p, uint32_t off, uint32_t f0) {
  if (off == 0) return 0;
  // F is a power of two <= 16 and f0 a multiple of it: the axes of the F frequencies are bits of one word
  const uint32_t axes = p.axis_of[f0 >> 4] >> (2 * (f0 & 15));
  uint32_t still = 0;
#pragma unroll
  for (int j = 0; j < F; ++j) still |= ((off >> ((axes >> (2 * j)) & 3u)) & 1u) << j;
  return still;
}

// x and y hold the F pairs (NeoX: two chunks of F elements; GPT-J: x holds the pairs, y is not used)
template <typename Tin, bool NEOX, int F, int VB>
__device__ __forceinline__ void turn(Chunk<VB>& x, Chunk<VB>& y, const float (&c)[F], const float (&s)[F], uint32_t still) {
  constexpr int ES = (int)sizeof(Tin);
  if constexpr (ES == 2 && (F % 2 == 0 || !NEOX)) {
    uint32_t* xw = reinterpret_cast<uint32_t*>(x.b);
    if constexpr (NEOX) {
      uint32_t* yw = reinterpret_cast<uint32_t*>(y.b);
#pragma unroll
      for (int j = 0; j < F; j += 2) {
        const uint32_t x0 = xw[j / 2], y0 = yw[j / 2];
        // two pairs at a time: the packed instructions round each half like the single ones
        const float2 u = unpack_pair<Tin>(x0), v = unpack_pair<Tin>(y0);
        const float2 c2 = make_float2(c[j], c[j + 1]), s2 = make_float2(s[j], s[j + 1]);
        const float2 vs = __fmul2_rn(v, s2);
        const float2 a = __ffma2_rn(u, c2, make_float2(-vs.x, -vs.y)), b = __ffma2_rn(v, c2, __fmul2_rn(u, s2));
        uint32_t x1 = pack_pair<Tin>(a.x, a.y), y1 = pack_pair<Tin>(b.x, b.y);
        if (still) {  // keep the halves that are not rotated
          const uint32_t keep = (((still >> j) & 1u) ? 0xFFFFu : 0u) | (((still >> (j + 1)) & 1u) ? 0xFFFF0000u : 0u);
          x1 = (x1 & ~keep) | (x0 & keep);
          y1 = (y1 & ~keep) | (y0 & keep);
        }
        xw[j / 2] = x1;
        yw[j / 2] = y1;
      }
    } else {
#pragma unroll
      for (int j = 0; j < F; ++j) {
        float u, v;
        unpack2<Tin>(xw[j], u, v);
        const uint32_t w = pack_pair<Tin>(__fmaf_rn(u, c[j], -__fmul_rn(v, s[j])), __fmaf_rn(v, c[j], __fmul_rn(u, s[j])));
        if (!((still >> j) & 1u)) xw[j] = w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < F; ++j) {
      unsigned char* px = NEOX ? x.b + j * ES : x.b + 2 * j * ES;
      unsigned char* py = NEOX ? y.b + j * ES : x.b + (2 * j + 1) * ES;
      const float u = to_f32<Tin>(px), v = to_f32<Tin>(py);
      if (!((still >> j) & 1u)) {
        put_float<Tin>(px, __fmaf_rn(u, c[j], -__fmul_rn(v, s[j])));
        put_float<Tin>(py, __fmaf_rn(v, c[j], __fmul_rn(u, s[j])));
      }
    }
  }
}

// Element offset of a cache slot.
__device__ __forceinline__ int64_t axes_slot_offset(const AxesParams& p, int64_t slot) {
  int64_t blk, off;
  split_slot(slot, p.block_size, p.bs_shift, blk, off);
  return blk * p.block_stride + off * p.page_stride;
}

// One item of the rotation is VEC elements of a head and, NeoX, their VEC partners; ALIGNED: they are one access each.
// The first rot_ctas CTAs rotate.  A CTA owns rows_per_cta consecutive (token, head) rows: a thread asks for its first
// items at once; meanwhile the CTA gathers the cosines and sines of its one to few tokens into shared memory,
// where all heads read them.  Measured, 16384 tokens x (64 + 8) heads x 128, three interleaved axes, bf16 (613 MB): 106 us
// = 5.8 TB/s.  CTAs of 256 threads 110 us, of 512 threads 143; four items per thread (256 threads) 124, the gather waits
// twice for memory and has to be spread over some work; each thread fetching cosines and sines of its own from the table
// rows of up to four axes, at 110 registers, 138.  The CTAs behind them move what is not rotated: elements from rot_dim on, and the values.
template <typename Tin, int KV, bool CACHE, bool NEOX, int VEC, bool ALIGNED>
__global__ void __launch_bounds__(kAxesThreads) rope_axes_kernel(const __grid_constant__ AxesParams p) {
  constexpr int ES = (int)sizeof(Tin);
  constexpr int VB = VEC * ES;
  constexpr int F = NEOX ? VEC : VEC / 2;
  constexpr int OUT_ES = (KV == KVC_KV_AUTO) ? ES : 1;
  extern __shared__ __align__(16) unsigned char axes_smem[];
  pdl_prologue();

  if (blockIdx.x < p.rot_ctas) {
    const uint32_t row0 = blockIdx.x * p.rows_per_cta;
    const uint32_t row_end = min(row0 + p.rows_per_cta, p.rows);
    const uint32_t items = (row_end - row0) * p.chunks;
    const uint32_t tok0 = p.div_heads.div(row0);
    const uint32_t tokens = p.div_heads.div(row_end - 1) - tok0 + 1;
    uint32_t* off = reinterpret_cast<uint32_t*>(axes_smem);
    unsigned char* turns = axes_smem + ((tokens * 4 + 15) & ~15u);

    struct Item {
      Chunk<VB> x, y;
      uint32_t tok, head, d0;
    };
    auto ask = [&](Item& it, uint32_t item) {
      if (item >= items) return;
      const uint32_t r = p.div_chunks.div(item);
      it.d0 = (item - r * p.chunks) * VEC;
      it.tok = p.div_heads.div(row0 + r);
      it.head = row0 + r - it.tok * p.num_heads;
      const Tin* src = it.head < p.num_q_heads
                           ? static_cast<const Tin*>(p.query) + it.tok * p.query_stride_t + it.head * p.query_stride_h
                           : static_cast<const Tin*>(p.key) + it.tok * p.key_stride_t +
                                 (it.head - p.num_q_heads) * p.key_stride_h;
      load_elements<Tin, ALIGNED>(it.x, src + it.d0);
      if constexpr (NEOX) load_elements<Tin, ALIGNED>(it.y, src + p.half + it.d0);
    };
    auto answer = [&](Item& it, uint32_t item) {
      if (item >= items) return;
      const uint32_t f0 = NEOX ? it.d0 : it.d0 / 2, t = it.tok - tok0;
      float c[F], s[F];
      if (sizeof(Tin) == 2 && p.table_f32)
        read_turns<float, F, ALIGNED>(reinterpret_cast<const float*>(turns) + t * p.rot_dim + f0, p.half, c, s);
      else
        read_turns<Tin, F, ALIGNED>(reinterpret_cast<const Tin*>(turns) + t * p.rot_dim + f0, p.half, c, s);
      turn<Tin, NEOX, F, VB>(it.x, it.y, c, s, still_mask<F>(p, off[t], f0));
      const bool is_query = it.head < p.num_q_heads;
      const uint32_t hk = it.head - p.num_q_heads;
      if (is_query || p.key_out != nullptr) {
        Tin* dst = is_query ? static_cast<Tin*>(p.query_out) + it.tok * p.qout_stride_t + it.head * p.qout_stride_h
                            : static_cast<Tin*>(p.key_out) + it.tok * p.kout_stride_t + hk * p.kout_stride_h;
        store_elements<ALIGNED, ES>(reinterpret_cast<char*>(dst + it.d0), it.x);
        if constexpr (NEOX) store_elements<ALIGNED, ES>(reinterpret_cast<char*>(dst + p.half + it.d0), it.y);
      }
      if constexpr (CACHE) {
        if (!is_query && it.tok < p.num_slot_tokens) {
          const int64_t slot = __ldg(p.slot_mapping + it.tok);
          if (slot >= 0) {
            ScaleCtx sc{};
            if constexpr (KV != KVC_KV_AUTO) sc = make_scale_ctx<Tin, KV>(p.k_scale);
            char* dst = static_cast<char*>(p.key_cache) + (axes_slot_offset(p, slot) + hk * p.head_stride + it.d0) * OUT_ES;
            Chunk<VEC * OUT_ES> out;
            convert_chunk<Tin, KV, VEC>(it.x, out, sc);
            store_elements<ALIGNED, OUT_ES>(dst, out);
            if constexpr (NEOX) {
              convert_chunk<Tin, KV, VEC>(it.y, out, sc);
              store_elements<ALIGNED, OUT_ES>(dst + static_cast<int64_t>(p.half) * OUT_ES, out);
            }
          }
        }
      }
    };

    // two items of a thread are being rotated while the next two are on their way
    Item it[4];
    ask(it[0], threadIdx.x);
    ask(it[1], threadIdx.x + kAxesThreads);
    for (uint32_t t = threadIdx.x; t < tokens; t += kAxesThreads) off[t] = 0;
    __syncthreads();
    if (sizeof(Tin) == 2 && p.table_f32) gather_turns(p, reinterpret_cast<float*>(turns), off, tok0, tokens);
    else gather_turns(p, reinterpret_cast<Tin*>(turns), off, tok0, tokens);
    __syncthreads();
    for (uint32_t item = threadIdx.x; item < items; item += 4 * kAxesThreads) {
      ask(it[2], item + 2 * kAxesThreads);
      ask(it[3], item + 3 * kAxesThreads);
      answer(it[0], item);
      answer(it[1], item + kAxesThreads);
      ask(it[0], item + 4 * kAxesThreads);
      ask(it[1], item + 5 * kAxesThreads);
      answer(it[2], item + 2 * kAxesThreads);
      answer(it[3], item + 3 * kAxesThreads);
    }
    return;
  }

  constexpr int CV = ALIGNED ? VEC : 1;
  const uint32_t item = (blockIdx.x - p.rot_ctas) * kAxesThreads + threadIdx.x;
  if (item >= p.copy_items) return;
  const uint32_t tok = p.div_copy.div(item);
  const uint32_t rem = item - tok * p.copy_per_token;
  Chunk<CV * ES> x;
  if (rem < p.seg_key) {  // query tail
    const uint32_t head = p.div_tail.div(rem);
    const uint32_t d0 = p.rot_dim + (rem - head * p.tail_chunks) * CV;
    load_chunk_inplace(x, static_cast<const Tin*>(p.query) + tok * p.query_stride_t + head * p.query_stride_h + d0);
    store_chunk(static_cast<Tin*>(p.query_out) + tok * p.qout_stride_t + head * p.qout_stride_h + d0, x, true);
    return;
  }
  uint32_t head, d0;
  const Tin* src;
  const bool is_value = rem >= p.seg_value;
  if (is_value) {
    const uint32_t j = rem - p.seg_value;
    head = p.div_value.div(j);
    d0 = (j - head * p.value_chunks) * CV;
    src = static_cast<const Tin*>(p.value) + tok * p.value_stride_t + head * p.value_stride_h + d0;
  } else {  // key tail
    const uint32_t j = rem - p.seg_key;
    head = p.div_tail.div(j);
    d0 = p.rot_dim + (j - head * p.tail_chunks) * CV;
    src = static_cast<const Tin*>(p.key) + tok * p.key_stride_t + head * p.key_stride_h + d0;
  }
  int64_t slot = -1;
  if constexpr (CACHE)
    if (tok < p.num_slot_tokens) slot = __ldg(p.slot_mapping + tok);
  const bool to_tensor = !is_value && p.key_out != nullptr && p.key_out != p.key;
  if (slot < 0 && !to_tensor) return;
  load_chunk_inplace(x, src);
  if (to_tensor) store_chunk(static_cast<Tin*>(p.key_out) + tok * p.kout_stride_t + head * p.kout_stride_h + d0, x, true);
  if constexpr (CACHE) {
    if (slot < 0) return;
    ScaleCtx sc{};
    if constexpr (KV != KVC_KV_AUTO) sc = make_scale_ctx<Tin, KV>(is_value ? p.v_scale : p.k_scale);
    Chunk<CV * OUT_ES> out;
    convert_chunk<Tin, KV, CV>(x, out, sc);
    store_chunk(static_cast<char*>(is_value ? p.value_cache : p.key_cache) +
                    (axes_slot_offset(p, slot) + head * p.head_stride + d0) * OUT_ES,
                out, true);
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
namespace {

struct AxesCall {
  AxesParams p;
  int64_t num_tokens, num_heads, num_kv_heads, head_size;
  const int64_t* sections;
  int64_t num_axes;
  bool neox, interleaved, cache;
  int in_dtype, table_dtype, kv_dtype;
};

int axes_fail(const char* text) { return fail(KVC_ERR_INVALID_ARG, std::string("multi_axis_rotary_embedding: ") + text); }

int check_axes(AxesCall& c) {
  AxesParams& p = c.p;
  if (c.in_dtype != KVC_IN_F32 && c.in_dtype != KVC_IN_F16 && c.in_dtype != KVC_IN_BF16)
    return fail(KVC_ERR_UNSUPPORTED, "multi_axis_rotary_embedding: unsupported tensor type code " + std::to_string(c.in_dtype));
  if (c.table_dtype != c.in_dtype && c.table_dtype != KVC_IN_F32)
    return fail(KVC_ERR_UNSUPPORTED, "multi_axis_rotary_embedding: cos_sin_cache must have the tensors' type or be fp32");
  if (c.num_tokens < 0 || c.num_heads < 0 || c.num_kv_heads < 0 || c.head_size <= 0) return axes_fail("negative size");
  if (p.rot_dim <= 0 || p.rot_dim % 2 || p.rot_dim > c.head_size)
    return axes_fail("rot_dim must be even and in (0, head_size]");
  if (p.rot_dim > 2 * kAxesMaxHalf)
    return fail(KVC_ERR_TOO_LARGE, "multi_axis_rotary_embedding: rot_dim is at most " + std::to_string(2 * kAxesMaxHalf));
  if (p.max_position <= 0) return axes_fail("max_position must be positive");
  if (c.head_size > 0x3FFFFFFFll || c.num_heads > 0x3FFFFFFFll || c.num_kv_heads > 0x3FFFFFFFll)
    return axes_fail("sizes out of range");
  if (c.num_axes < 1 || c.num_axes > kAxesMax) return axes_fail("between 1 and 4 position axes are supported");
  if (!c.sections) return axes_fail("the sections of the axes must be given");
  const int64_t half = p.rot_dim / 2;
  int64_t sum = 0;
  for (int64_t a = 0; a < c.num_axes; ++a) {
    if (c.sections[a] < 0 || c.sections[a] > half) return axes_fail("a section is negative or larger than rot_dim / 2");
    sum += c.sections[a];
  }
  if (sum != half) return axes_fail("the sections must add up to rot_dim / 2");
  if (c.interleaved)
    for (int64_t a = 1; a < c.num_axes; ++a)
      if (c.sections[a] > 0 && (c.sections[a] - 1) * c.num_axes + a >= half)
        return axes_fail("an interleaved section does not fit into rot_dim / 2");
  for (int64_t a = 0, i = 0; a < c.num_axes; ++a)
    for (int64_t n = 0; n < c.sections[a]; ++n, ++i)
      if (!c.interleaved) p.axis_of[i >> 4] |= static_cast<uint32_t>(a) << (2 * (i & 15));
  if (c.interleaved)
    for (int64_t i = 0; i < half; ++i) {
      const int64_t a = i % c.num_axes;
      if (a > 0 && i / c.num_axes < c.sections[a]) p.axis_of[i >> 4] |= static_cast<uint32_t>(a) << (2 * (i & 15));
    }
  if (c.num_tokens == 0) return KVC_OK;
  const int es = in_elem_size(c.in_dtype);
  if (!p.positions || !p.cos_sin_cache || (c.num_heads > 0 && (!p.query || !p.query_out)) || (c.num_kv_heads > 0 && !p.key))
    return axes_fail("positions, query, key (when it has heads) and cos_sin_cache must be non-NULL");
  if (!aligned(p.positions, 8)) return axes_fail("positions must be 8-byte aligned");
  if (!aligned(p.query, es) || !aligned(p.key, es) || !aligned(p.query_out, es) || !aligned(p.key_out, es) ||
      !aligned(p.value, es) || !aligned(p.cos_sin_cache, in_elem_size(c.table_dtype)))
    return axes_fail("tensors are not aligned to their element size");
  return KVC_OK;
}

// The widest item whose accesses every address, stride and length of the call allows: 16 bytes, 4 bytes, or
// (vec_aligned false) single elements.  The table's address does not matter: its elements are gathered one by one.
int axes_vec(const AxesCall& c, bool& vec_aligned) {
  const AxesParams& p = c.p;
  const int es = in_elem_size(c.in_dtype);
  const int out_es = c.kv_dtype == KVC_KV_AUTO ? es : 1;
  const int64_t half = p.half, tail = c.head_size - p.rot_dim;
  const int widths[2] = {16 / es, 2};
  for (int i = 0; i < (es == 2 ? 2 : 1); ++i) {
    const int vec = widths[i];
    const int64_t vb = static_cast<int64_t>(vec) * es;
    const int f = c.neox ? vec : vec / 2;
    bool ok = half % f == 0 && tail % vec == 0;
    auto rows = [&](const void* base, int64_t st, int64_t sh) {
      return aligned(base, vb) && (st * es) % vb == 0 && (sh * es) % vb == 0;
    };
    if (c.neox) ok = ok && (half * es) % vb == 0;
    if (c.num_heads > 0)
      ok = ok && rows(p.query, p.query_stride_t, p.query_stride_h) && rows(p.query_out, p.qout_stride_t, p.qout_stride_h);
    if (c.num_kv_heads > 0) {
      ok = ok && rows(p.key, p.key_stride_t, p.key_stride_h);
      if (p.key_out) ok = ok && rows(p.key_out, p.kout_stride_t, p.kout_stride_h);
    }
    if (c.cache) {
      const int64_t ob = static_cast<int64_t>(vec) * out_es;
      ok = ok && rows(p.value, p.value_stride_t, p.value_stride_h) && c.head_size % vec == 0;
      ok = ok && aligned(p.key_cache, ob) && aligned(p.value_cache, ob) && (p.block_stride * out_es) % ob == 0 &&
           (p.page_stride * out_es) % ob == 0 && (p.head_stride * out_es) % ob == 0 && (half * out_es) % (c.neox ? ob : 1) == 0;
    }
    if (ok) {
      vec_aligned = true;
      return vec;
    }
  }
  vec_aligned = false;
  return c.neox ? 1 : 2;
}

// A CTA's shared memory: at most kAxesItems * kAxesThreads items of at least two frequencies' worth of cosines and sines
// each, in fp32, and a flag per token (one kv head, small heads, an fp32 table: 68 KB).
constexpr int kAxesMaxSmem = 72 * 1024;

cudaError_t launch_axes_kernel(void (*kernel)(const AxesParams), dim3 grid, int smem, const AxesParams& p, cudaStream_t st) {
  if (smem > kAxesMaxSmem) return cudaErrorInvalidValue;
  if (smem > 48 * 1024) {  // always to the same value: calls of other threads and captured ones may need other amounts
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAxesMaxSmem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kAxesThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename Tin, int KV, bool CACHE, bool NEOX>
cudaError_t launch_axes_vec(int vec, bool vec_aligned, const AxesParams& p, dim3 grid, int smem, cudaStream_t st) {
  constexpr int ES = (int)sizeof(Tin);
  if (!vec_aligned) return launch_axes_kernel(rope_axes_kernel<Tin, KV, CACHE, NEOX, NEOX ? 1 : 2, false>, grid, smem, p, st);
  if constexpr (ES == 2)
    if (vec == 2) return launch_axes_kernel(rope_axes_kernel<Tin, KV, CACHE, NEOX, 2, true>, grid, smem, p, st);
  return launch_axes_kernel(rope_axes_kernel<Tin, KV, CACHE, NEOX, 16 / ES, true>, grid, smem, p, st);
}

template <typename Tin>
cudaError_t launch_axes(const AxesCall& c, int vec, bool vec_aligned, dim3 grid, int smem, cudaStream_t st) {
  const AxesParams& p = c.p;
  if (!c.cache)
    return c.neox ? launch_axes_vec<Tin, KVC_KV_AUTO, false, true>(vec, vec_aligned, p, grid, smem, st)
                  : launch_axes_vec<Tin, KVC_KV_AUTO, false, false>(vec, vec_aligned, p, grid, smem, st);
  switch (c.kv_dtype) {
    case KVC_KV_AUTO:
      return c.neox ? launch_axes_vec<Tin, KVC_KV_AUTO, true, true>(vec, vec_aligned, p, grid, smem, st)
                    : launch_axes_vec<Tin, KVC_KV_AUTO, true, false>(vec, vec_aligned, p, grid, smem, st);
    case KVC_KV_FP8_E4M3:
      return c.neox ? launch_axes_vec<Tin, KVC_KV_FP8_E4M3, true, true>(vec, vec_aligned, p, grid, smem, st)
                    : launch_axes_vec<Tin, KVC_KV_FP8_E4M3, true, false>(vec, vec_aligned, p, grid, smem, st);
    default:
      return c.neox ? launch_axes_vec<Tin, KVC_KV_FP8_E5M2, true, true>(vec, vec_aligned, p, grid, smem, st)
                    : launch_axes_vec<Tin, KVC_KV_FP8_E5M2, true, false>(vec, vec_aligned, p, grid, smem, st);
  }
}

int axes_impl(AxesCall& c, cudaStream_t st) {
  AxesParams& p = c.p;
  p.half = p.rot_dim / 2;
  if (!c.p.query_out) {  // in place
    p.query_out = const_cast<void*>(p.query);
    p.qout_stride_t = p.query_stride_t;
    p.qout_stride_h = p.query_stride_h;
  }
  if (int rc = check_axes(c)) return rc;
  if (c.cache) {
    if (c.kv_dtype != KVC_KV_AUTO && c.kv_dtype != KVC_KV_FP8_E4M3 && c.kv_dtype != KVC_KV_FP8_E5M2)
      return fail(KVC_ERR_UNSUPPORTED, "Unsupported data type of kv cache: code " + std::to_string(c.kv_dtype));
    if (p.block_size <= 0) return axes_fail("block_size must be positive");
    if (p.num_slot_tokens < 0 || p.num_slot_tokens > c.num_tokens) return axes_fail("num_slot_tokens must be in [0, num_tokens]");
  }
  if (c.num_tokens == 0 || c.num_heads + c.num_kv_heads == 0) return KVC_OK;
  const int es = in_elem_size(c.in_dtype), out_es = c.kv_dtype == KVC_KV_AUTO ? es : 1;
  if (c.cache) {
    if (c.num_kv_heads == 0) return axes_fail("the cache write needs key heads");
    if (!p.value || !p.key_cache || !p.value_cache || (p.num_slot_tokens > 0 && !p.slot_mapping))
      return axes_fail("value, key_cache, value_cache and slot_mapping must be non-NULL");
    if (c.kv_dtype != KVC_KV_AUTO && (!p.k_scale || !p.v_scale))
      return axes_fail("k_scale and v_scale must be non-NULL for an fp8 cache");
    if (!aligned(p.slot_mapping, 8) || !aligned(p.key_cache, out_es) || !aligned(p.value_cache, out_es))
      return axes_fail("slot_mapping and the caches must be aligned to their element size");
  }
  p.bs_shift = c.cache ? pow2_shift(p.block_size) : -1;
  p.table_f32 = c.table_dtype != c.in_dtype;
  p.num_q_heads = static_cast<uint32_t>(c.num_heads);
  const int64_t heads = c.num_heads + c.num_kv_heads;
  p.num_heads = static_cast<uint32_t>(heads);
  bool vec_aligned;
  const int vec = axes_vec(c, vec_aligned);
  const int64_t chunks = p.half / (c.neox ? vec : vec / 2);
  const bool q_tail = p.query_out != p.query, k_tail = c.cache || (p.key_out && p.key_out != p.key);
  const int64_t cv = vec_aligned ? vec : 1;
  const int64_t tail = (c.head_size - p.rot_dim) / cv;
  const int64_t rot_per_token = heads * chunks;
  const int64_t seg_key = q_tail ? c.num_heads * tail : 0;
  const int64_t seg_value = seg_key + (k_tail ? c.num_kv_heads * tail : 0);
  const int64_t copy_per_token = seg_value + (c.cache ? c.num_kv_heads * (c.head_size / cv) : 0);
  if (rot_per_token + copy_per_token >= (1ll << 30)) return axes_fail("heads * head_size too large");
  p.chunks = static_cast<uint32_t>(chunks);
  p.tail_chunks = static_cast<uint32_t>(tail);
  p.value_chunks = static_cast<uint32_t>(c.head_size / cv);
  p.seg_key = static_cast<uint32_t>(seg_key);
  p.seg_value = static_cast<uint32_t>(seg_value);
  p.copy_per_token = static_cast<uint32_t>(copy_per_token);
  p.div_chunks = FastDiv(p.chunks);
  p.div_heads = FastDiv(p.num_heads);
  p.div_half = FastDiv(static_cast<uint32_t>(p.half));
  p.div_copy = FastDiv(copy_per_token ? p.copy_per_token : 1);
  p.div_tail = FastDiv(tail ? p.tail_chunks : 1);
  p.div_value = FastDiv(p.value_chunks);

  const AxesParams base = p;
  const int64_t most = rot_per_token > copy_per_token ? rot_per_token : copy_per_token;
  int64_t step = ((1ll << 31) - kAxesThreads) / most;
  auto moved = [&](const void* q, int64_t elements, int size) {
    return q ? const_cast<char*>(static_cast<const char*>(q)) + elements * size : nullptr;
  };
  for (int64_t t0 = 0; t0 < c.num_tokens; t0 += step) {
    const int64_t nt = c.num_tokens - t0 < step ? c.num_tokens - t0 : step;
    p.positions = base.positions + t0;
    p.query = moved(base.query, t0 * p.query_stride_t, es);
    p.query_out = moved(base.query_out, t0 * p.qout_stride_t, es);
    p.key = moved(base.key, t0 * p.key_stride_t, es);
    p.key_out = moved(base.key_out, t0 * p.kout_stride_t, es);
    p.value = moved(base.value, t0 * p.value_stride_t, es);
    p.slot_mapping = base.slot_mapping ? base.slot_mapping + t0 : nullptr;
    p.num_slot_tokens = base.num_slot_tokens - t0;  // may be <= 0: no slots in this launch
    p.rows = static_cast<uint32_t>(nt * heads);
    // one item per thread where the call has few, so that it spreads over the SMs
    const int64_t per_cta = nt * rot_per_token < 148 * 2 * kAxesItems * kAxesThreads ? kAxesThreads : kAxesItems * kAxesThreads;
    p.rows_per_cta = static_cast<uint32_t>(chunks < per_cta ? per_cta / chunks : 1);
    p.copy_items = static_cast<uint32_t>(nt * copy_per_token);
    p.rot_ctas = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
    // tokens whose rows meet in one CTA: their flags and their cosines and sines
    const int64_t met = (p.rows_per_cta + heads - 2) / heads + 1;
    const int smem = static_cast<int>(((met * 4 + 15) & ~15ll) + met * p.rot_dim * (p.table_f32 ? 4 : es));
    const dim3 grid(p.rot_ctas + (p.copy_items + kAxesThreads - 1) / kAxesThreads);
    cudaError_t e;
    if (c.in_dtype == KVC_IN_F32) e = launch_axes<float>(c, vec, vec_aligned, grid, smem, st);
    else if (c.in_dtype == KVC_IN_F16) e = launch_axes<__half>(c, vec, vec_aligned, grid, smem, st);
    else e = launch_axes<__nv_bfloat16>(c, vec, vec_aligned, grid, smem, st);
    if (e != cudaSuccess)
      return fail(KVC_ERR_CUDA, std::string("multi_axis_rotary_embedding launch failed: ") + cudaGetErrorString(e));
  }
  return KVC_OK;
}

}  // namespace
}  // namespace kvc

// ---------------------------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------------------------
extern "C" {

KVC_API int kvc_multi_axis_rotary_embedding(
    const int64_t* positions, const int64_t* axis_sections, const void* query, const void* key, void* query_out,
    void* key_out, const void* cos_sin_cache, int64_t num_axes, int64_t position_stride, int64_t num_tokens,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_size, int64_t rot_dim, int64_t max_position,
    int64_t query_stride_t, int64_t query_stride_h, int64_t key_stride_t, int64_t key_stride_h,
    int64_t query_out_stride_t, int64_t query_out_stride_h, int64_t key_out_stride_t, int64_t key_out_stride_h,
    int is_neox, int interleaved, int in_dtype, int table_dtype, void* stream) {
  kvc::AxesCall c{};
  c.p.positions = positions;
  c.p.query = query;
  c.p.key = key;
  c.p.query_out = query_out;
  c.p.key_out = key_out ? key_out : const_cast<void*>(key);
  c.p.cos_sin_cache = cos_sin_cache;
  c.p.position_stride = position_stride;
  c.p.max_position = max_position;
  c.p.rot_dim = rot_dim < 0 || rot_dim > 0x3FFFFFFFll ? 0 : static_cast<int32_t>(rot_dim);
  c.p.query_stride_t = query_stride_t;
  c.p.query_stride_h = query_stride_h;
  c.p.key_stride_t = key_stride_t;
  c.p.key_stride_h = key_stride_h;
  c.p.qout_stride_t = query_out_stride_t;
  c.p.qout_stride_h = query_out_stride_h;
  c.p.kout_stride_t = key_out ? key_out_stride_t : key_stride_t;
  c.p.kout_stride_h = key_out ? key_out_stride_h : key_stride_h;
  c.num_tokens = num_tokens;
  c.num_heads = num_heads;
  c.num_kv_heads = key ? num_kv_heads : 0;
  c.head_size = head_size;
  c.sections = axis_sections;
  c.num_axes = num_axes;
  c.neox = is_neox != 0;
  c.interleaved = interleaved != 0;
  c.in_dtype = in_dtype;
  c.table_dtype = table_dtype;
  return kvc::axes_impl(c, static_cast<cudaStream_t>(stream));
}

KVC_API int kvc_multi_axis_rotary_embedding_and_cache_flash(
    const int64_t* positions, const int64_t* axis_sections, const void* query, void* key, const void* value,
    void* query_out, const void* cos_sin_cache, void* key_cache, void* value_cache, const int64_t* slot_mapping,
    int64_t num_axes, int64_t position_stride, int64_t num_tokens, int64_t num_slot_tokens, int64_t num_heads,
    int64_t num_kv_heads, int64_t head_size, int64_t rot_dim, int64_t max_position, int64_t block_size,
    int64_t query_stride_t, int64_t query_stride_h, int64_t key_stride_t, int64_t key_stride_h, int64_t value_stride_t,
    int64_t value_stride_h, int64_t query_out_stride_t, int64_t query_out_stride_h, int64_t block_stride,
    int64_t page_stride, int64_t head_stride, int is_neox, int interleaved, int write_back_key, int in_dtype,
    int table_dtype, int kv_dtype, const float* k_scale, const float* v_scale, void* stream) {
  kvc::AxesCall c{};
  c.p.positions = positions;
  c.p.query = query;
  c.p.key = key;
  c.p.query_out = query_out;
  c.p.key_out = write_back_key ? key : nullptr;
  c.p.cos_sin_cache = cos_sin_cache;
  c.p.value = value;
  c.p.key_cache = key_cache;
  c.p.value_cache = value_cache;
  c.p.slot_mapping = slot_mapping;
  c.p.k_scale = k_scale;
  c.p.v_scale = v_scale;
  c.p.position_stride = position_stride;
  c.p.max_position = max_position;
  c.p.num_slot_tokens = num_slot_tokens;
  c.p.rot_dim = rot_dim < 0 || rot_dim > 0x3FFFFFFFll ? 0 : static_cast<int32_t>(rot_dim);
  c.p.query_stride_t = query_stride_t;
  c.p.query_stride_h = query_stride_h;
  c.p.key_stride_t = key_stride_t;
  c.p.key_stride_h = key_stride_h;
  c.p.value_stride_t = value_stride_t;
  c.p.value_stride_h = value_stride_h;
  c.p.qout_stride_t = query_out_stride_t;
  c.p.qout_stride_h = query_out_stride_h;
  c.p.kout_stride_t = key_stride_t;
  c.p.kout_stride_h = key_stride_h;
  c.p.block_stride = block_stride;
  c.p.page_stride = page_stride;
  c.p.head_stride = head_stride;
  c.p.block_size = block_size;
  c.num_tokens = num_tokens;
  c.num_heads = num_heads;
  c.num_kv_heads = num_kv_heads;
  c.head_size = head_size;
  c.sections = axis_sections;
  c.num_axes = num_axes;
  c.neox = is_neox != 0;
  c.interleaved = interleaved != 0;
  c.cache = true;
  c.in_dtype = in_dtype;
  c.table_dtype = table_dtype;
  c.kv_dtype = kv_dtype;
  return kvc::axes_impl(c, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
