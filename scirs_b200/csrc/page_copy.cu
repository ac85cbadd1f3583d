// Copies of cache pages: the first counts[i] slots of page src[i] go to page dst[i], in the K and the
// V pool of every layer, in one launch. Forked sequences get their own copy of a page that two
// sequences would write, and a fragmented pool is made compact, with it.
//
// A page is one contiguous run of block_size * Hkv * HD elements in each pool, so this is a plain
// memory copy of many runs: 2 x bytes of traffic and nothing to compute. The page ids and the pools'
// addresses travel as kernel parameters (no table in device memory has to be written first, and a
// captured graph keeps them); a CTA takes a chunk of 256 x U 16-byte vectors of one run at a time, U of
// them in flight per thread. Measured: 680 pages of 32 KB in 32 pools (1.43 GB read and written) 249 us,
// 5.7 TB/s, 0.87 of a plain device copy's rate; 64 partly filled pages in 48 pools (107 MB) 21 us; 8 in 24
// pools 2.7 us on the device, 8 us a call, bound by the call on the host.
//
// Reference parity: scirs2-neural/src/inference/block_manager.rs:196-280 (page chains and the shared
// prefix cache; pages are never copied there).
#include "host_common.h"

namespace scirs {
namespace pages {

constexpr int kThreads = 256;

template <int MOVES, int BUFS>
struct Args {
  uint4* buf[BUFS];
  int src[MOVES], dst[MOVES], vecs[MOVES];  // vecs: 16-byte vectors to copy
  int moves, bufs, chunks;                  // chunks of a whole page
  long page_vecs;
};

template <int MOVES, int BUFS, int U>
__global__ void __launch_bounds__(kThreads) copy_kernel(const __grid_constant__ Args<MOVES, BUFS> a) {
  const long units = (long)a.bufs * a.moves * a.chunks;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = (int)(u % a.chunks);
    const long r = u / a.chunks;
    const int i = (int)(r % a.moves);
    uint4* base = a.buf[r / a.moves];
    const uint4* s = base + (long)a.src[i] * a.page_vecs;
    uint4* d = base + (long)a.dst[i] * a.page_vecs;
    const long v0 = (long)c * (kThreads * U) + threadIdx.x;
    uint4 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (v0 + j * kThreads < a.vecs[i]) x[j] = __ldg(s + v0 + j * kThreads);
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (v0 + j * kThreads < a.vecs[i]) d[v0 + j * kThreads] = x[j];
  }
}

// Returns how many launches it took.
template <int MOVES, int BUFS, int U>
int64_t launch(const std::vector<torch::Tensor>& bufs, const int* src, const int* dst, const int* counts, int n,
            int slot_vecs, int block_size) {
  const int dev = bufs[0].get_device();
  Args<MOVES, BUFS> a;
  a.page_vecs = (long)slot_vecs * block_size;
  a.chunks = (int)((a.page_vecs + kThreads * U - 1) / (kThreads * U));
  int64_t launches = 0;
  for (size_t b0 = 0; b0 < bufs.size(); b0 += BUFS) {
    a.bufs = (int)std::min<size_t>(BUFS, bufs.size() - b0);
    for (int b = 0; b < a.bufs; ++b) a.buf[b] = reinterpret_cast<uint4*>(bufs[b0 + b].data_ptr());
    for (int m0 = 0; m0 < n; m0 += MOVES) {
      a.moves = std::min(MOVES, n - m0);
      for (int i = 0; i < a.moves; ++i) {
        a.src[i] = src[m0 + i];
        a.dst[i] = dst[m0 + i];
        a.vecs[i] = slot_vecs * (counts != nullptr ? counts[m0 + i] : block_size);
      }
      const long units = (long)a.bufs * a.moves * a.chunks;
      const int grid = (int)std::min<long>(units, 8L * num_sms(dev));
      copy_kernel<MOVES, BUFS, U><<<grid, kThreads, 0, cur_stream()>>>(a);
      SCIRS_CHECK_LAUNCH();
      ++launches;
    }
  }
  return launches;
}

}  // namespace pages

// bufs: the pools ([num_pages, block_size, Hkv, HD], all of one shape and type on one device);
// src / dst / counts: int32 on the host. Every index is checked here, before the launch. Returns the launches made.
int64_t page_copy(std::vector<torch::Tensor> bufs, torch::Tensor src, torch::Tensor dst,
                  c10::optional<torch::Tensor> counts) {
  TORCH_CHECK(!bufs.empty(), "page_copy: no pools");
  const torch::Tensor& f = bufs[0];
  TORCH_CHECK(f.is_cuda() && f.dim() == 4, "pools: CUDA [num_pages, block_size, Hkv, HD]");
  const int64_t num_pages = f.size(0), bs = f.size(1);
  const int64_t slot_bytes = f.size(2) * f.size(3) * f.element_size();
  TORCH_CHECK(slot_bytes > 0 && slot_bytes % 16 == 0, "a token's keys must be a multiple of 16 bytes");
  TORCH_CHECK(bs * slot_bytes / 16 < (1LL << 31) && num_pages < (1LL << 31), "page or pool too large");
  for (const auto& t : bufs)
    TORCH_CHECK(t.device() == f.device() && t.sizes() == f.sizes() && t.scalar_type() == f.scalar_type() &&
                    t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                "pools must be contiguous, 16-byte aligned and alike in device, shape and type");
  const int64_t n = src.numel();
  auto host = [&](const torch::Tensor& t, const char* what) {
    TORCH_CHECK(!t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 && t.numel() == n,
                what, ": int32 [", num(n), "] on the host");
    return t.data_ptr<int>();
  };
  const int *s = host(src, "src"), *d = host(dst, "dst");
  const int* c = counts.has_value() && counts->defined() ? host(*counts, "counts") : nullptr;
  std::vector<uint8_t> written(num_pages, 0);
  for (int64_t i = 0; i < n; ++i) {
    TORCH_CHECK(s[i] >= 0 && s[i] < num_pages && d[i] >= 0 && d[i] < num_pages, "page ", num(s[i]), " -> ", num(d[i]),
                " is outside the pool of ", num(num_pages));
    TORCH_CHECK(c == nullptr || (c[i] >= 0 && c[i] <= bs), "a count of ", num(c ? c[i] : 0), " of ", num(bs),
                " slots");
    TORCH_CHECK(!written[d[i]], "page ", num(d[i]), " is written twice");
    written[d[i]] = 1;
  }
  for (int64_t i = 0; i < n; ++i) TORCH_CHECK(!written[s[i]], "page ", num(s[i]), " is both read and written");
  if (n == 0) return 0;
  c10::cuda::CUDAGuard guard(f.get_device());
  return pages::launch<1024, 256, 4>(bufs, s, d, c, (int)n, (int)(slot_bytes / 16), (int)bs);
}

}  // namespace scirs
