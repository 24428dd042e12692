// Pages between the fp32 pool and the int8 one (pool_attention.hip has the layouts, int8_rows.h the rows' form).
#include "int8_rows.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kThreads = 256;
constexpr int kD = 128;
constexpr int kRows = 16;    // rows of a workgroup: four of each wave
constexpr int kAtOnce = 5;   // pairs of heads whose loads are under way together

// Bound by memory: 24 pages over 12 layers in 106 us, 4.5 TB/s read and written; back, 5 half pages in 10 us.  Half a wave has
// a head's row, four values a lane: 512 contiguous bytes of the fp32 pool and 128 of the int8 one a head.  Pairs count as if
// one were converted after the other: rows of a page that a later pair writes too are left to it.
template <bool kQuantize>
__global__ void __launch_bounds__(kThreads) k_convert_pages(ConvertPages p) {
  __shared__ int later;
  const int pair = (int)blockIdx.x, lane = lane_id(), part = (int)blockIdx.z * kRows;
  const int from = ldg(p.src + pair), to = ldg(p.dst + pair);
  const int src_pages = kQuantize ? p.fp32_pages : p.int8_pages, dst_pages = kQuantize ? p.int8_pages : p.fp32_pages;
  if (from < 0 || from >= src_pages || to < 0 || to >= dst_pages) return;
  if (threadIdx.x == 0) later = 0;
  __syncthreads();
  for (int i = pair + 1 + (int)threadIdx.x; i < p.count; i += kThreads) {
    const int f = ldg(p.src + i);
    if (ldg(p.dst + i) == to && f >= 0 && f < src_pages) atomicMax(&later, p.rows != nullptr ? ldg(p.rows + i) : p.page_size);
  }
  __syncthreads();
  const int begin = max(later, part);
  const int end = min(min(part + kRows, p.page_size), p.rows != nullptr ? ldg(p.rows + pair) : p.page_size);
  const int half = lane / 32, c = lane % 32;
  for (int r = begin + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave); r < end; r += kThreads / kWave) {
    const int64_t at = (int64_t)blockIdx.y * p.page_size + r;  // blockIdx.y: k or v, and the layer
    const int64_t of_page = 2 * (int64_t)p.layers * p.page_size;
    float* wide = p.fp32 + ((kQuantize ? from : to) * of_page + at) * p.heads * kD;
    char* slot = p.int8 + ((kQuantize ? to : from) * of_page + at) * p.slot_bytes;
    float* scales = (float*)(slot + p.heads * kD);
    for (int h0 = half; h0 < p.heads; h0 += 2 * kAtOnce) {
      if constexpr (kQuantize) {
        f32x4 x[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          x[i] = *(const UOCR_GLOBAL f32x4*)(wide + min(h0 + 2 * i, p.heads - 1) * kD + 4 * c);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          uint32_t most = max(max(abs_bits(x[i].x), abs_bits(x[i].y)), max(abs_bits(x[i].z), abs_bits(x[i].w)));
          for (int off = 16; off >= 1; off /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, off, kWave));
          const float s = row_scale(most);
          const uint32_t q = to_int8x4(x[i].x, x[i].y, x[i].z, x[i].w, s);
          if (h0 + 2 * i < p.heads) {
            stg((uint32_t*)(slot + (h0 + 2 * i) * kD) + c, q);
            if (c == 0) stg(scales + h0 + 2 * i, s);
          }
        }
      } else {
        uint32_t q[kAtOnce];
        float s[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int h = min(h0 + 2 * i, p.heads - 1);
          q[i] = ldg((const uint32_t*)(slot + h * kD) + c);
          s[i] = ldg(scales + h);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (h0 + 2 * i < p.heads)
            *(UOCR_GLOBAL f32x4*)(wide + (h0 + 2 * i) * kD + 4 * c) =
                f32x4{i8_to_f32<0>((int)q[i]), i8_to_f32<1>((int)q[i]), i8_to_f32<2>((int)q[i]), i8_to_f32<3>((int)q[i])} * s[i];
      }
    }
  }
}

}  // namespace

hipError_t launch_convert_pages(const ConvertPages& p, bool quantize, hipStream_t s) {
  if (p.count == 0) return hipSuccess;
  const dim3 grid((unsigned)p.count, (unsigned)(2 * p.layers), (unsigned)((p.page_size + kRows - 1) / kRows));
  if (quantize)
    UOCR_LAUNCH("quantize_pages", k_convert_pages<true>, grid, dim3(kThreads), 0, s, p);
  else
    UOCR_LAUNCH("dequantize_pages", k_convert_pages<false>, grid, dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace uocr
