// Launchers of the paged decode attention (paged_decode.cuh).
#include <algorithm>
#include <mutex>

#include "paged_decode.cuh"

namespace q6w {
namespace paged {

constexpr int kMaxPerSm = 4;  // CTAs an SM at most: the workspace is laid out for that many

size_t decode_workspace(int hd) {
  const size_t ctas = (size_t)sm_count() * kMaxPerSm;
  return ctas * 2 * state_floats(hd, 8) * sizeof(float) + ctas * sizeof(int4);
}

template <int HD, typename KT, int R>
static int32_t launch(DecodeArgs a, cudaStream_t st) {
  using S = DecodeShape<HD, KT, R>;
  auto kern = decode_kernel<HD, KT, R>;
  constexpr int smem = kDecodeWarps * S::WARP;
  // per device: CTAs an SM, with the kernel's shared memory granted once
  static std::mutex mu;
  static int per_sm[64] = {0};
  int dev = 0, occ = 0;
  Q6W_CUDA_TRY(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!per_sm[dev & 63]) {
      Q6W_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      Q6W_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kDecodeThreads, smem));
      per_sm[dev & 63] = std::min(std::max(occ, 1), kMaxPerSm);
    }
    occ = per_sm[dev & 63];
  }
  const int64_t most = (int64_t)a.b.n * a.b.kv_heads * a.HB * std::max<int64_t>(1, (a.b.max_len + S::CH - 1) / S::CH);
  const int grid = (int)std::min<int64_t>((int64_t)sm_count() * occ, most);
  kern<<<grid, kDecodeThreads, smem, st>>>(a);
  Q6W_LAUNCH_CHECK("decode_kernel");
  merge_kernel<HD, R><<<dim3(grid, (R * HD + 127) / 128), 128, 0, st>>>(a);
  Q6W_LAUNCH_CHECK("merge_kernel");
  return Q6W_OK;
}

template <int HD, typename KT>
static int32_t launch_r(const DecodeArgs& a, cudaStream_t st) {
  if (a.per > 4) return launch<HD, KT, 8>(a, st);
  if (a.per > 2) return launch<HD, KT, 4>(a, st);
  if (a.per > 1) return launch<HD, KT, 2>(a, st);
  return launch<HD, KT, 1>(a, st);
}

int32_t decode_attention(const DecodeArgs& a, int hd, bool half, cudaStream_t st) {
  switch (hd) {
    case 16: return half ? launch_r<16, __half>(a, st) : launch_r<16, float>(a, st);
    case 32: return half ? launch_r<32, __half>(a, st) : launch_r<32, float>(a, st);
    case 64: return half ? launch_r<64, __half>(a, st) : launch_r<64, float>(a, st);
    default: return half ? launch_r<128, __half>(a, st) : launch_r<128, float>(a, st);
  }
}

}  // namespace paged
}  // namespace q6w
