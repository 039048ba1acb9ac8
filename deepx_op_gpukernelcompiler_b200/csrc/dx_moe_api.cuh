// dx_moe_api.cuh — host side of the mixture-of-experts layer: argument checks,
// workspace layout, TMA descriptors and the two launches.  Part of dx_api.cu (it
// uses that file's helpers).
#pragma once

#include "dx_moe.cuh"

namespace {

using dx::MoeParams;
using dx::MoeRouterParams;
using dx::MoeShape;

struct MoeLayout {
  size_t h = 0, partials = 0, counters = 0, bytes = 0;  // offsets; h holds hi, then lo
  int64_t chosen = 0;                                   // most experts that can be chosen
  int num_counters = 0;
};

MoeLayout moe_layout(int64_t T, int64_t H, int64_t E, int64_t top, int ctas) {
  MoeLayout l;
  l.chosen = std::min<int64_t>(E, T * top);
  auto place = [&l](size_t bytes) {
    const size_t at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  l.h = place(static_cast<size_t>(l.chosen * T * H) * 2 * 2);
  l.partials = place(static_cast<size_t>(ctas) * dx::kMoeSlots * 2 * static_cast<size_t>(T) * 128 *
                     sizeof(float));
  l.num_counters = 2 * ctas + 1;
  l.counters = place(static_cast<size_t>(l.num_counters) * sizeof(int));
  return l;
}

// 16-bit [E][rows][cols] with pitches in elements, a [1 x 64 x 64] box.
int make_tmap_expert(CUtensorMap* m, const void* ptr, CUtensorMapDataType dt, int64_t cols,
                     int64_t rows, int64_t E, int64_t ld, int64_t ld_expert, const char* name) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                        static_cast<cuuint64_t>(E)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(ld_expert) * 2};
  cuuint32_t box[3] = {64, 64, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = g_encode(m, dt, 3, const_cast<void*>(ptr), dims, strides, box, es,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(DX_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name,
                static_cast<int>(r));
  return DX_OK;
}

int moe_validate(const dx_moe_args* a) {
  if (a == nullptr) return fail(DX_ERR_INVALID_ARGUMENT, "moe: NULL arguments");
  if (a->dtype == DX_DTYPE_F32)
    return fail(DX_ERR_UNSUPPORTED, "moe: fp16 or bf16 (the kernel is a 16-bit tensor-core one)");
  if (a->dtype != DX_DTYPE_F16 && a->dtype != DX_DTYPE_BF16)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: unknown dtype %d", a->dtype);
  if (a->act < DX_ACT_NONE || a->act > DX_ACT_SILU)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: unknown activation %d", a->act);
  if (a->T < 0 || a->D < 1 || a->H < 1 || a->E < 1 || a->top_k < 1)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: T >= 0 and D, H, E, top_k >= 1");
  if (a->T > dx::kMoeMaxT || a->E > dx::kMoeMaxE || a->top_k > dx::kMoeMaxTop)
    return fail(DX_ERR_UNSUPPORTED, "moe: at most %d tokens, %d experts and top_k %d, got %lld, %lld, %lld",
                dx::kMoeMaxT, dx::kMoeMaxE, dx::kMoeMaxTop, (long long)a->T, (long long)a->E,
                (long long)a->top_k);
  if (a->top_k > a->E)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: top_k=%lld of E=%lld experts", (long long)a->top_k,
                (long long)a->E);
  if (a->D % 8 != 0 || a->H % 8 != 0 || a->D > 65536 || a->H > 65536)
    return fail(DX_ERR_UNSUPPORTED, "moe: D and H must be multiples of 8 up to 65536, got %lld, %lld",
                (long long)a->D, (long long)a->H);
  if (a->T == 0) return DX_OK;
  if (a->X == nullptr || a->Wr == nullptr || a->Wg == nullptr || a->Wu == nullptr ||
      a->Wo == nullptr || a->Y == nullptr || a->ids == nullptr || a->weights == nullptr)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: X, a weight, Y, ids or weights is NULL");
  if (a->ldx < a->D || a->ldwr < a->E || a->ldy < a->D || (a->R != nullptr && a->ldr < a->D) ||
      a->ldg < a->H || a->ldu < a->H || a->ldo < a->D)
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: a pitch is below its row length");
  auto bad = [](const void* p, int64_t ld, int64_t lde) {
    return !aligned16(p) || ld % 8 != 0 || lde % 8 != 0;
  };
  if (bad(a->X, a->ldx, 0) || bad(a->Wg, a->ldg, a->ldg_expert) ||
      bad(a->Wu, a->ldu, a->ldu_expert) || bad(a->Wo, a->ldo, a->ldo_expert))
    return fail(DX_ERR_UNSUPPORTED,
                "moe: X and the expert weights need 16-byte-aligned pointers and pitches");
  if (a->E > 1 && (a->ldg_expert < a->ldg * a->D || a->ldu_expert < a->ldu * a->D ||
                   a->ldo_expert < a->ldo * a->H))
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: an expert's pitch is below its matrix");
  if (!element_aligned(2, a->Wr, a->br, a->bg, a->bu, a->bo, a->R, a->Y) ||
      !element_aligned(4, a->ids, a->weights))
    return fail(DX_ERR_INVALID_ARGUMENT, "moe: a pointer is not aligned to its elements");
  return DX_OK;
}

template <int MN, typename T>
int launch_moe_experts(const dx_moe_args& a, int dev, int ctas, const MoeLayout& l,
                       cudaStream_t stream) {
  using S = MoeShape;
  auto kern = dx::moe_experts_kernel<MN, T>;
  const int mn = static_cast<int>((a.T + 15) / 16 * 16);
  const int pairs = static_cast<int>(a.T * a.top_k);
  const int stages = S::max_stages(mn, pairs);
  int rc = ensure_smem_attr(dev, reinterpret_cast<const void*>(kern), 227 * 1024, true);
  if (rc) return rc;
  char* const ws = static_cast<char*>(a.workspace);
  MoeParams p{};
  p.T = static_cast<int>(a.T);
  p.D = static_cast<int>(a.D);
  p.H = static_cast<int>(a.H);
  p.E = static_cast<int>(a.E);
  p.top = static_cast<int>(a.top_k);
  p.act = a.act;
  p.kb_d = static_cast<int>((a.D + 63) / 64);
  p.nt_h = static_cast<int>((a.H + 127) / 128);
  p.kb_h = static_cast<int>((a.H + 63) / 64);
  p.nt_d = static_cast<int>((a.D + 255) / 256);
  p.mn = mn;
  p.stages = stages;
  p.ids = a.ids;
  p.weights = a.weights;
  p.bg = a.bg;
  p.bu = a.bu;
  p.bo = a.bo;
  p.residual = a.R;
  p.ldr = a.ldr;
  p.Y = a.Y;
  p.ldy = a.ldy;
  p.h_hi = ws + l.h;
  p.h_lo = ws + l.h + static_cast<size_t>(l.chosen * a.T * a.H) * 2;
  p.partials = reinterpret_cast<float*>(ws + l.partials);
  p.counters = reinterpret_cast<int*>(ws + l.counters);
  const CUtensorMapDataType dt = tma_dtype(a.dtype);
  CUtensorMap tG, tU, tO, tX, tHi, tLo;
  if ((rc = make_tmap_expert(&tG, a.Wg, dt, a.H, a.D, a.E, a.ldg, a.ldg_expert, "Wg"))) return rc;
  if ((rc = make_tmap_expert(&tU, a.Wu, dt, a.H, a.D, a.E, a.ldu, a.ldu_expert, "Wu"))) return rc;
  if ((rc = make_tmap_expert(&tO, a.Wo, dt, a.D, a.H, a.E, a.ldo, a.ldo_expert, "Wo"))) return rc;
  if ((rc = make_tmap_2d(&tX, a.X, dt, a.D, a.T, a.ldx, 64, mn, CU_TENSOR_MAP_SWIZZLE_128B, "X")))
    return rc;
  if ((rc = make_tmap_2d(&tHi, p.h_hi, dt, a.H, l.chosen * a.T, a.H, 64, mn,
                         CU_TENSOR_MAP_SWIZZLE_128B, "h")))
    return rc;
  if ((rc = make_tmap_2d(&tLo, p.h_lo, dt, a.H, l.chosen * a.T, a.H, 64, mn,
                         CU_TENSOR_MAP_SWIZZLE_128B, "h")))
    return rc;
  const int smem = S::smem_bytes(mn, stages, pairs);
  set_plan_ints("moe T=%d mn=%d stages=%d grid=%d smem=%d", p.T, mn, stages, ctas, smem);
  // Cooperative: the CTAs wait for one another, so all of them or none are placed.
  cudaLaunchAttribute attr[3];
  cudaLaunchConfig_t cfg = launch_config(ctas, S::THREADS, smem, stream, 1, attr);
  attr[cfg.numAttrs].id = cudaLaunchAttributeCooperative;
  attr[cfg.numAttrs].val.cooperative = 1;
  ++cfg.numAttrs;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tG, tU, tO, tX, tHi, tLo, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch moe_experts_kernel");
  return DX_OK;
}

template <typename T>
int launch_moe(const dx_moe_args& a, int dev, int ctas, const MoeLayout& l, cudaStream_t stream) {
  MoeRouterParams r{};
  r.X = a.X;
  r.Wr = a.Wr;
  r.br = a.br;
  r.ldx = a.ldx;
  r.ldwr = a.ldwr;
  r.T = static_cast<int>(a.T);
  r.D = static_cast<int>(a.D);
  r.E = static_cast<int>(a.E);
  r.top = static_cast<int>(a.top_k);
  r.renormalize = a.renormalize;
  r.ids = a.ids;
  r.weights = a.weights;
  r.counters = reinterpret_cast<int*>(static_cast<char*>(a.workspace) + l.counters);
  r.num_counters = l.num_counters;
  const int groups = (r.T + dx::kRouterTokens - 1) / dx::kRouterTokens;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_config(groups * dx::kRouterTokens, dx::kRouterThreads, 0, stream,
                                         dx::kRouterTokens, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, dx::moe_router_kernel<T>, r);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch moe_router_kernel");
  if (a.T <= 16) return launch_moe_experts<16, T>(a, dev, ctas, l, stream);
  if (a.T <= 32) return launch_moe_experts<32, T>(a, dev, ctas, l, stream);
  return launch_moe_experts<64, T>(a, dev, ctas, l, stream);
}

}  // namespace

extern "C" {

size_t dx_moe_workspace_size(int64_t T, int64_t H, int64_t E, int64_t top_k) {
  if (T < 1 || T > dx::kMoeMaxT || H < 1 || H > 65536 || E < 1 || E > dx::kMoeMaxE || top_k < 1 ||
      top_k > std::min<int64_t>(E, dx::kMoeMaxTop))
    return 0;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || device_sms(dev, &sms) != DX_OK) {
    (void)cudaGetLastError();
    return 0;
  }
  return moe_layout(T, H, E, top_k, sms).bytes;
}

int dx_moe(const dx_moe_args* a, void* stream) {
  t_last_error.clear();
  int rc = moe_validate(a);
  if (rc) return rc;
  if (a->T == 0) return DX_OK;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int sms = 0, ctas = 0;
  if ((rc = device_sms(dev, &sms))) return rc;
  const MoeLayout l = moe_layout(a->T, a->H, a->E, a->top_k, sms);
  if (a->workspace == nullptr || a->workspace_bytes < l.bytes ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
    return fail(DX_ERR_WORKSPACE, "moe needs a 256-byte-aligned workspace of %zu bytes", l.bytes);
  if ((rc = stream_sms(s, dev, &ctas))) return rc;
  if ((rc = install_status_mirror(dev, s))) return rc;
  if ((rc = check_status_mirror(dev))) return rc;
  if (!load_encode_fn())
    return fail(DX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  return a->dtype == DX_DTYPE_F16 ? launch_moe<__half>(*a, dev, ctas, l, s)
                                  : launch_moe<__nv_bfloat16>(*a, dev, ctas, l, s);
}

}  // extern "C"
