// Attention whose results leave in blocks of 32 (mx.h), the rows of an output projection held in 4 bits, without a quantisation behind it.  A
// result is rounded to bfloat16 first, as it is where the two are launches of their own, so that the blocks are theirs bit for bit.
//
// Decode steps: the merge of the splits writes them.  Beside the heads' workgroups there are some for the columns from nq * D to the rows' padding, which leave
// zeros.  A row whose result is there already, because its keys had one wave or its splits met inside a workgroup, is read back from `out`.
#pragma once
#include "attention_stream.h"
#include "mx.h"

namespace arle {

struct MergeBlocks {
  uint8_t* elements;
  uint8_t* scales;
  int bits, padded;     // padded: columns of a row, a multiple of 512
};

template <int BITS>
__device__ __forceinline__ void leave_blocks(const MergeBlocks& b, int row, int col, float4 v) {     // of a wave's first D / 4 lanes
  const uint32_t code = mx_code<BITS>(mx_lanes_max<8>(mx_max4(v)));
  mx_store4<BITS>(b.elements + static_cast<int64_t>(row) * (BITS == kMx8 ? b.padded : b.padded / 2), col, mx_pack4<BITS>(v, code));
  if (col % kMxBlock == 0) b.scales[static_cast<int64_t>(row) * (b.padded / kMxBlock) + col / kMxBlock] = static_cast<uint8_t>(code);
}

// Single decoded tokens: segment s is row s.  ws_o null: every row is read back.
template <int BITS>
__global__ __launch_bounds__(kMergeWaves* kWave) void attn_merge_blocks_kernel(
    const float* __restrict__ ws_o, const float* __restrict__ ws_ml, const uint16_t* __restrict__ out, int64_t o_stride,
    const int* __restrict__ seg_row0, int nq, int nkv, int D, int splits, const float* __restrict__ sink, float out_scale,
    const int* __restrict__ plan, MergeBlocks blocks) {
  const int seg = blockIdx.x, head = blockIdx.y;
  if (head >= nq || ws_o == nullptr || (plan != nullptr && plan[2 * seg + 1] == 1)) {     // the whole workgroup
    const int d0 = 4 * threadIdx.x;
    if (d0 >= D) return;
    uint2 w = {0, 0};
    if (head < nq) w = *reinterpret_cast<const uint2*>(out + seg * o_stride + head * D + d0);
    leave_blocks<BITS>(blocks, seg, head * D + d0,
                       float4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)});
    return;
  }
  const auto rounded = [](float v) { return __uint_as_float(static_cast<uint32_t>(f32_to_bf16_bits(v)) << 16); };
  attn_merge_body(ws_o, ws_ml, seg_row0, 1, 0, nq, nkv, D, splits, sink, out_scale, plan, [&](int row, int h, int d0, float4 o) {
    leave_blocks<BITS>(blocks, row, h * D + d0, float4{rounded(o.x), rounded(o.y), rounded(o.z), rounded(o.w)});
  });
}

// Portions: a row's block in two lanes, lane j with columns 8 q + e of it and lane j + 32 with 8 q + 4 + e, as pairs of bfloat16.
// (Head_dim 128 and rows of whole 512 columns, so that there is no padding.)
template <int BITS>
__device__ __forceinline__ void leave_block(const AttnArgs& a, int row, int col, int h, const uint2 (&w)[4]) {
  float4 v[4];
  uint32_t most = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    v[q] = float4{__uint_as_float(w[q].x << 16), __uint_as_float(w[q].x & 0xffff0000u), __uint_as_float(w[q].y << 16), __uint_as_float(w[q].y & 0xffff0000u)};
    most = max(most, mx_max4(v[q]));
  }
  const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
  const uint32_t code = mx_code<BITS>(max(both[0], both[1]));
  const int64_t width = static_cast<int64_t>(a.nq) * a.D;
#pragma unroll
  for (int q = 0; q < 4; ++q) mx_store4<BITS>(a.blocks + row * (BITS == kMx8 ? width : width / 2), col + 8 * q + 4 * h, mx_pack4<BITS>(v[q], code));
  if (h == 0) a.block_scales[row * (width / kMxBlock) + col / kMxBlock] = static_cast<uint8_t>(code);
}

}  // namespace arle
