// C ABI of the weight gradient of the grouped GEMM: argument checks, tensor maps, launch.
#include "dg_host.h"
#include "dg_grouped_wgrad.cuh"

namespace {

using namespace dg;
using namespace dg::host;

template <int S>
struct Stages { static constexpr int value = S; };

template <int CL, int S, bool kSegments, bool kSplit = false>
int launch_wgrad(const dg_weight_grad_args* a, WgradParams p, const DeviceInfo& dev, cudaStream_t stream) {
  auto kernel = grouped_wgrad_kernel<CL, S, kSegments, kSplit>;
  const int cluster = kSplit ? p.split : CL;
  constexpr int BT = 128 * CL;
  p.n_tiles = (p.N + BT - 1) / BT;
  p.k_tiles = (p.K + BT - 1) / BT;
  const long long items = (long long)p.G * p.n_tiles * p.k_tiles;
  if (items > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  const int smem = WgradSmem<S, wg_wide(kSegments, kSplit) ? 8 : 4>::total(p.G, p.m_blocks);
  if (smem > dev.max_smem) return DG_ERR_TOO_LARGE;

  CUtensorMap tm_dy, tm_x, tm_d;
  // Without rows nothing is loaded; the maps then describe one row that is never read.
  const uint64_t rows = p.M > 0 ? p.M : 1;
  // [64-column blocks][rows][64 columns]; when N is no multiple of 64 the last block of a row would
  // reach into the next one, and behind the last row, so dy is then [rows][columns].
  p.dy_blocks = p.N % 64 == 0;
  auto operand = [&](CUtensorMap* map, const void* base, int cols, bool blocks) {
    const uint64_t dims[3] = {blocks ? 64u : (uint64_t)cols, rows, (uint64_t)cols / 64};
    const uint64_t strides[2] = {(uint64_t)cols * 2, 128};
    const uint32_t box[3] = {64u, 64u, 2u};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, blocks ? 3 : 2, p.M > 0 ? base : a->dw, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  };
  int rc = operand(&tm_dy, a->dy, p.N, p.dy_blocks);
  if (rc == DG_OK) rc = operand(&tm_x, a->x, p.K, true);
  const uint64_t es = p.f32 ? 4 : 2;
  const uint64_t d_dims[3] = {64u, (uint64_t)p.N, (uint64_t)p.G * (p.K / 64)};
  const uint64_t d_str[2] = {64 * es, 64 * es * p.N};
  const uint32_t d_box[3] = {p.f32 ? 32u : 64u, 32u, 1u};
  if (rc == DG_OK)
    rc = encode_map(&tm_d, p.f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a->dw, d_dims, d_str,
                    d_box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != DG_OK) return rc;

  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(wg_threads(kSegments, kSplit), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;

  // Once per device: opt in to the shared-memory size and ask how many clusters fit at once.
  static std::mutex mu;
  static int max_units[kMaxDevices] = {0};
  int devid = 0;
  cudaGetDevice(&devid);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (max_units[devid] == 0) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dev.max_smem);
      if (e != cudaSuccess) return cuda_fail(e);
      if (!kSplit) {
        cudaLaunchConfig_t q = cfg;
        q.gridDim = dim3(dev.sm_count / CL * CL, 1, 1);
        q.dynamicSmemBytes = dev.max_smem;
        int n = 0;
        e = cudaOccupancyMaxActiveClusters(&n, kernel, &q);
        if (e != cudaSuccess) return cuda_fail(e);
        if (n < 1) return DG_ERR_TOO_LARGE;
        max_units[devid] = n < dev.sm_count / CL ? n : dev.sm_count / CL;
      } else {
        max_units[devid] = 0x7fffffff / 8;  // a cluster for every tile: none waits for another
      }
    }
  }
  const long long units = items < max_units[devid] ? items : max_units[devid];
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * units), 1, 1);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tm_dy, tm_x, tm_d, p);
  if (e != cudaSuccess) return cuda_fail(e);
  count_launches(1);
  return DG_OK;
}

}  // namespace

extern "C" {

int dg_grouped_weight_grad(const dg_weight_grad_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (a->num_groups < 1 || a->m_total < 0 || a->n < 16 || a->n % 16 != 0 || a->k < 64 || a->k % 64 != 0) return DG_ERR_BAD_SHAPE;
  if (a->out_kind != DG_OUT_BF16 && a->out_kind != DG_OUT_F32) return DG_ERR_BAD_ARGUMENT;
  if (a->accumulate != 0 && a->out_kind != DG_OUT_F32) return DG_ERR_BAD_ARGUMENT;  // sums are kept in 32 bits
  if (a->tile != 0 && a->tile != 128 && a->tile != 256 && a->tile != 1) return DG_ERR_BAD_ARGUMENT;
  if (a->num_groups > DG_MAX_GROUPS || a->m_total > DG_MAX_CONTIG_ROWS) return DG_ERR_TOO_LARGE;
  if ((long long)a->num_groups * (a->k / 64) > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  if (!a->dw || (a->m_total > 0 && (!a->dy || !a->x || !a->m_indices))) return DG_ERR_NULL_POINTER;
  if (!aligned16(a->dy) || !aligned16(a->x) || !aligned16(a->dw)) return DG_ERR_BAD_ALIGNMENT;
  if (a->m_total == 0 && a->accumulate) return DG_OK;
  const long long dw_bytes = (a->out_kind == DG_OUT_F32 ? 4LL : 2LL) * a->num_groups * a->n * a->k;
  if (overlap(a->dw, dw_bytes, a->dy, 2LL * a->m_total * a->n) || overlap(a->dw, dw_bytes, a->x, 2LL * a->m_total * a->k) ||
      overlap(a->dw, dw_bytes, a->m_indices, 4LL * a->m_total))
    return DG_ERR_BAD_ARGUMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  WgradParams p{};
  p.G = a->num_groups;
  p.M = a->m_total;
  p.N = a->n;
  p.K = a->k;
  p.m_blocks = (a->m_total + 127) / 128;
  p.m_indices = a->m_indices;
  p.dy = static_cast<const __nv_bfloat16*>(a->dy);
  p.x = static_cast<const __nv_bfloat16*>(a->x);
  p.status = a->status;
  p.f32 = a->out_kind == DG_OUT_F32;
  p.add = a->accumulate != 0;
  p.dw = a->dw;
  p.whole_blocks = a->whole_blocks != 0;
  p.segment = p.f32 ? kWgSegment : DG_MAX_CONTIG_ROWS / 128;
  // 256 x 256 tiles move half the operand bytes per product, which pays when a group has rows enough
  // and there are tiles enough; else 128 x 128 ones, whose epilogues are shorter and which reach more
  // SMs.  Measured, 128 against 256, us: 32 groups of 1024 rows, 4096 x 7168: 2018 / 1469; 256 of 128 rows,
  // 1024 x 1792: 244 / 322; 16 of 64 rows, 4096 x 1024: 41 / 50; 32 of 300 rows, 1024 x 512: 24.5 /
  // 24.2; 4 of 1000 rows, 1024 x 1024 (64 tiles of 256): 17.0 / 14.9; 8 of 2000 rows, 512 x 512 (32
  // tiles): 19.1 / 22.4.
  const long long rows = p.M / p.G;
  const long long items256 = (long long)p.G * ((p.N + 255) / 256) * ((p.K + 255) / 256);
  const long long items128 = (long long)p.G * ((p.N + 127) / 128) * ((p.K + 127) / 128);
  const int tile = a->tile != 0 ? a->tile : (rows >= 320 && items256 >= 48 ? 256 : 128);
  // Fewer 128 x 128 tiles than a half of the SMs and a long way along the rows: a tile is split, as
  // often as there are SMs for it and four row blocks for every part.  us without and with: 1 group of
  // 16000 rows, 256 x 64: 74.8 / 20.1; of 8000 rows, 512 x 768: 40.6 / 19.4; of 2000 rows, 128 x 128: 14.3 /
  // 10.7; but 2 of 1000 rows, 256 x 256: 10.3 / 11.1.
  int split = 1;
  while (rows >= 1536 && split < 8 && items128 * split * 2 <= dev->sm_count && rows >= 128LL * 4 * split * 2) split *= 2;
  if (a->tile == 1) split = 4;  // (asked for)
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool splits = (a->tile == 0 && tile == 128 && split > 1) || a->tile == 1;
  p.split = split;
  auto go = [&](auto stages) {
    constexpr int S = decltype(stages)::value;
    if (splits) return launch_wgrad<1, S, true, true>(a, p, *dev, st);
    // (fp32: a stage's room goes to the strips of four more epilogue warps)
    if (p.f32) return tile == 256 ? launch_wgrad<2, S - 1, true>(a, p, *dev, st) : launch_wgrad<1, S - 1, true>(a, p, *dev, st);
    return tile == 256 ? launch_wgrad<2, S, false>(a, p, *dev, st) : launch_wgrad<1, S, false>(a, p, *dev, st);
  };
  // the table of very many rows takes the room of a ring stage
  if (WgradSmem<kWgStages, 4>::total(p.G, p.m_blocks) <= dev->max_smem) return go(Stages<kWgStages>{});
  return go(Stages<kWgStages - 1>{});
}

}  // extern "C"
