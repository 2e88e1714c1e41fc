// Launchers of the logits head, one translation unit per type of hidden states.
#pragma once

#include "ets_w4.h"

namespace ets_host {

// How the weights are laid out: what picks an instantiation besides the hidden states' type.
struct HeadForm {
  int groups_per_chunk;  // 4, 2 or 1
  int scale_bytes;       // 4 or 2
  bool zeros;
};

hipError_t launch_head_f32(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream);
hipError_t launch_head_f16(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream);
hipError_t launch_head_bf16(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream);

template <int XT, int GPC, int SB, bool ZEROS>
hipError_t launch_head(const ets::HeadParams& p, hipStream_t stream) {
  constexpr int NT = 4;
  const dim3 grid((p.tiles + NT - 1) / NT, (p.rows + 15) / 16);
  hipLaunchKernelGGL((ets::head_stream_kernel<XT, GPC, SB, ZEROS, NT>), grid, dim3(ets::kHeadBlock), 0, stream, p);
  return hipGetLastError();
}

template <int XT, int GPC, int MT, int NT, int WV, int WK>
hipError_t launch_tiles(const ets::HeadParams& p, hipStream_t stream) {
  const int64_t vocab_blocks = (p.tiles + WV * NT - 1) / (WV * NT), row_blocks = (p.rows + 16 * MT - 1) / (16 * MT);
  hipLaunchKernelGGL((ets::head_tile_kernel<XT, GPC, MT, NT, WV, WK>), dim3(static_cast<uint32_t>((vocab_blocks + 7) / 8 * 8 * row_blocks)),
                     dim3(64 * WV * WK), 0, stream, p);
  return hipGetLastError();
}

template <int XT, int GPC, int MT>
hipError_t launch_tiles(const ets::HeadParams& p, hipStream_t stream) {
  // 256 vocabulary entries a workgroup where that makes at least one for each of the 256 CUs; otherwise 128, with twice
  // the waves behind each other along the columns.
  return p.tiles >= 256 * 16 ? launch_tiles<XT, GPC, MT, 4, 4, 1>(p, stream) : launch_tiles<XT, GPC, MT, 2, 4, 2>(p, stream);
}

template <int XT, int GPC>
hipError_t launch_head(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream) {
  if (p.rows > 16) {
    if (p.rows <= 32 || XT == ets::kDtypeFloat) return launch_tiles<XT, GPC, 2>(p, stream);
    return launch_tiles<XT, GPC, XT == ets::kDtypeFloat ? 2 : 4>(p, stream);
  }
  if (f.scale_bytes == 4) return f.zeros ? launch_head<XT, GPC, 4, true>(p, stream) : launch_head<XT, GPC, 4, false>(p, stream);
  return f.zeros ? launch_head<XT, GPC, 2, true>(p, stream) : launch_head<XT, GPC, 2, false>(p, stream);
}

template <int XT>
hipError_t launch_head(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream) {
  switch (f.groups_per_chunk) {
    case 4: return launch_head<XT, 4>(p, f, stream);
    case 2: return launch_head<XT, 2>(p, f, stream);
    default: return launch_head<XT, 1>(p, f, stream);
  }
}

}  // namespace ets_host
