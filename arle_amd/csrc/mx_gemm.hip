// Products of microscaled rows with a weight in 4 bits:  C[M,N] = X[M,K] . W[N,K]^T, X in e4m3 or e2m1, W in e2m1, both in
// blocks of 32 along K with a power of two each (mx.h).  v_mfma_scale takes elements and scales as they are: an operand is 32
// elements a lane and one scale byte a lane, the sum of a block's products times the two scales, added in 32 bits.
//
// W is laid out once as operand tiles of 16 columns x 128 k, [ceil(N/16)][K/128][64][16 bytes], lane 16 g + i: W[16 t + i][128 s + 32 g
// .. + 31], one contiguous kilobyte a wave and load; its scales as [ceil(N/16)][ceil(K/512)][64] words, byte s % 4 of lane 16 g + i
// for that lane's block of tile s.  K is padded with zeros to a multiple of 256 on both sides.
//
// With W as the first operand (rows of the result are W's columns) a lane ends up with four neighbouring columns of one row.
// Operand layouts of the second operand's lane (row i, group g): e2m1 32 neighbouring k from 32 g on, as the first; e4m3 16 neighbouring
// from 16 g on and 16 from half the instruction's k + 16 g on.  Scales go by blocks of 32 neighbouring k in either case:
// lane group g's byte is the scale of block g.  With e4m3 the instruction aligns the products of 8 neighbouring k to the largest of
// them and drops what is under 2^-13 of it (measured with pairs of products); everything behind that is 32 bits wide.  That is 2^-9
// of what rounding to e4m3 has taken from a number before.
#include "mx.h"

#include <type_traits>

namespace arle {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMxF32 = 0, kMxBf16 = 1, kMxGate8 = 2, kMxGate4 = 3;   // what leaves: sums, or silu(gate) * up in blocks

struct MxArgs {
  const uint8_t* x;
  int64_t ldx;            // bytes between rows of elements
  const uint8_t* xs;
  int64_t ldxs;
  const uint8_t* w;
  const uint32_t* ws;
  void* out;
  int64_t ldo, split_stride;
  uint8_t* out_scales;
  int64_t ldos;
  int M, N, n_tiles, k_tiles;
  int per_split;          // steps of K that one workgroup walks
  int vec;                // rows of `out` take whole 16-byte stores
  int m_blocks, n_blocks;
};

__device__ __forceinline__ mx_i32x8 mx_operand4(u32x4 v) {
  return mx_i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}
__device__ __forceinline__ mx_i32x8 mx_operand8(u32x4 a, u32x4 b) {
  return mx_i32x8{static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]),
                  static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
}
__device__ __forceinline__ float mx_silu_mul(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

template <int EPI>
__device__ __forceinline__ void mx_store_sums(const MxArgs& a, int split, int row, int n, mx_f32x4 v) {
  if (row >= a.M || n >= a.N) return;
  if constexpr (EPI == kMxF32) {
    float* o = static_cast<float*>(a.out) + split * a.split_stride + static_cast<int64_t>(row) * a.ldo + n;
    if (a.vec && n + 4 <= a.N) {
      *reinterpret_cast<mx_f32x4*>(o) = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) o[e] = v[e];
  } else {
    bf16* o = static_cast<bf16*>(a.out) + static_cast<int64_t>(row) * a.ldo + n;
    if (a.vec && n + 4 <= a.N) {
      *reinterpret_cast<uint2*>(o) = uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) o[e] = from_float<bf16>(v[e]);
  }
}

// ---- few rows: W is streamed once
//
// A workgroup owns CT column tiles and a part of K (blockIdx.y); its WAVES waves take the part's tiles in turn and add their sums
// through LDS in the order of the waves.  X comes from the caches, straight into operands.
template <int BITS, int RT, int CT, int WAVES, int U, int EPI>
__global__ __launch_bounds__(WAVES* kWave) void mx_gemm_rows_kernel(const MxArgs a) {
  constexpr bool kGate = EPI == kMxGate8 || EPI == kMxGate4;
  static_assert(!kGate || CT == 4, "a block of 32 results is two tiles of gate and two of up columns");
  constexpr int kSub = 17, kTile = 4 * kSub;      // places of a tile's four columns x 16 rows, padded against bank conflicts
  __shared__ mx_f32x4 parts[WAVES][RT * CT][kTile];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int ct0 = blockIdx.x * CT, k_tiles = a.k_tiles, k_groups = (k_tiles + 3) / 4;
  const int begin = blockIdx.y * a.per_split, end = min(begin + a.per_split, k_tiles);

  const uint8_t* wp[CT];
  const uint32_t* wsp[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int64_t tile = min(ct0 + c, a.n_tiles - 1);
    wp[c] = a.w + tile * k_tiles * 1024 + lane * 16;
    wsp[c] = a.ws + tile * k_groups * 64 + lane;
  }
  const uint8_t* xp[RT];
  const uint8_t* xsp[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t row = min(16 * r + i, a.M - 1);
    xp[r] = a.x + row * a.ldx + 16 * g;
    xsp[r] = a.xs + row * a.ldxs;
  }
  struct Step {
    u32x4 w[CT], x[RT][BITS == kMx8 ? 2 : 1];
    uint32_t ws[CT], xs[RT];
  };
  auto load = [&](int t, Step& s) {
    t = min(t, end - 1);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      s.w[c] = *reinterpret_cast<const u32x4*>(wp[c] + static_cast<int64_t>(t) * 1024);
      s.ws[c] = wsp[c][(t >> 2) * 64];
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if constexpr (BITS == kMx8) {
        s.x[r][0] = *reinterpret_cast<const u32x4*>(xp[r] + static_cast<int64_t>(t) * 128);
        s.x[r][1] = *reinterpret_cast<const u32x4*>(xp[r] + static_cast<int64_t>(t) * 128 + 64);
      } else {
        s.x[r][0] = *reinterpret_cast<const u32x4*>(xp[r] + static_cast<int64_t>(t) * 64);
      }
      s.xs[r] = *reinterpret_cast<const uint32_t*>(xsp[r] + 4 * t);
    }
  };
  mx_f32x4 acc[RT][CT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[r][c] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int t, const Step& s) {
    if (t >= end) return;     // the same in all lanes
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      mx_i32x8 xo;
      if constexpr (BITS == kMx8)
        xo = mx_operand8(s.x[r][0], s.x[r][1]);
      else
        xo = mx_operand4(s.x[r][0]);
      const int xscale = static_cast<int>(s.xs[r] >> (8 * g));
#pragma unroll
      for (int c = 0; c < CT; ++c)
        acc[r][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand4(s.w[c]), xo, acc[r][c], 4, BITS == kMx8 ? 0 : 4, 0,
                                                                     static_cast<int>(s.ws[c] >> (8 * (t & 3))), 0, xscale);
    }
  };
  Step now[U], next[U];
  int t = begin + wave;
#pragma unroll
  for (int u = 0; u < U; ++u) load(t + u * WAVES, now[u]);
  while (t < end) {
#pragma unroll
    for (int u = 0; u < U; ++u) load(t + (U + u) * WAVES, next[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) multiply(t + u * WAVES, now[u]);
    t += U * WAVES;
    if (t >= end) break;
#pragma unroll
    for (int u = 0; u < U; ++u) load(t + (U + u) * WAVES, now[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) multiply(t + u * WAVES, next[u]);
    t += U * WAVES;
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) parts[wave][r * CT + c][g * kSub + i] = acc[r][c];
  __syncthreads();

  auto sum = [&](int tile, int at) {
    mx_f32x4 s = parts[0][tile][at];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += parts[w][tile][at];
    return s;
  };
  if constexpr (kGate) {
    for (int item = tid; item < RT * 16 * 8; item += WAVES * kWave) {     // (row, four of 32 results): eight lanes a block
      const int row = item >> 3, q = item & 7, tile = (row >> 4) * CT + 2 * (q >> 2), at = (q & 3) * kSub + (row & 15);
      const mx_f32x4 gate = sum(tile, at), up = sum(tile + 1, at);
      const float4 v = {mx_silu_mul(gate[0], up[0]), mx_silu_mul(gate[1], up[1]), mx_silu_mul(gate[2], up[2]), mx_silu_mul(gate[3], up[3])};
      constexpr int kBits = EPI == kMxGate8 ? kMx8 : kMx4;
      const uint32_t code = mx_code<kBits>(mx_lanes_max<8>(mx_max4(v)));
      if (row < a.M) {
        mx_store4<kBits>(static_cast<uint8_t*>(a.out) + row * a.ldo, 32 * blockIdx.x + 4 * q, mx_pack4<kBits>(v, code));
        if (q == 0) a.out_scales[row * a.ldos + blockIdx.x] = static_cast<uint8_t>(code);
      }
    }
  } else {
    for (int item = tid; item < RT * 16 * CT * 4; item += WAVES * kWave) {
      const int row = item / (CT * 4), q = item % (CT * 4);
      mx_store_sums<EPI>(a, blockIdx.y, row, 16 * ct0 + 4 * q, sum((row >> 4) * CT + (q >> 2), (q & 3) * kSub + (row & 15)));
    }
  }
}

// ---- many rows
//
// A workgroup of RW x CW waves owns 32 MT RW rows and 32 TN CW columns; a wave 32 MT rows and 32 TN columns.  A step is 128 bytes of
// every row of X: 128 k of e4m3, 256 of e2m1.  X goes through registers into LDS, rows of 128 bytes whose 16-byte pieces are
// exchanged by the row (piece c of row r at c ^ (r % 8)), so that neither the lanes that park a row nor the lanes that read a
// column of pieces share banks; two stages.  W goes straight from its tiles into operands, PD steps ahead.
template <int BITS, int MT, int TN, int RW, int CW, int PD, int EPI>
__global__ __launch_bounds__(RW* CW* kWave) void mx_gemm_tiles_kernel(const MxArgs a) {
  constexpr bool kGate = EPI == kMxGate8 || EPI == kMxGate4;
  static_assert(!kGate || TN == 2, "a block of 32 results is two tiles of 16 gate and 16 up columns");
  static_assert(PD % 2 == 0, "the stage alternates inside a round");
  constexpr int kThreads = RW * CW * kWave, kRows = 32 * MT * RW;
  constexpr int KT = BITS == kMx8 ? 1 : 2, KK = 2 * KT;      // tiles of 128 k and halves of 64 k in a step
  constexpr int kStage = kRows * (128 + 4 * KT);
  constexpr int XH = kRows * 8 / kThreads;
  static_assert(XH * kThreads == kRows * 8 && kRows <= kThreads * 2, "whole pieces a thread");
  constexpr int XS = (kRows + kThreads - 1) / kThreads;      // rows whose scales a thread parks
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31, h = lane >> 5;
  const int wr = wave / CW, wc = wave % CW;

  // workgroup -> (row block, column block): an XCD's workgroups one behind the other, eight row blocks of a column block side by side
  const int total = a.m_blocks * a.n_blocks, per_xcd = (total + 7) / 8;
  const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per_xcd || id >= total) return;   // the whole workgroup
  const int group = id / (8 * a.n_blocks), first = group * 8, rows_here = min(8, a.m_blocks - first), in = id - group * 8 * a.n_blocks;
  const int mb = first + in % rows_here, nb = in / rows_here;
  const int m0 = mb * kRows, n0 = (nb * CW + wc) * (32 * TN);
  const int k_tiles = a.k_tiles, k_groups = (k_tiles + 3) / 4, steps = k_tiles / KT;
  const int s_begin = blockIdx.y * a.per_split, n_steps = min(a.per_split, steps - s_begin);

  const uint8_t* wptr[TN];
  const uint32_t* wsptr[TN];
#pragma unroll
  for (int tn = 0; tn < TN; ++tn) {
    const int64_t tile = min(n0 / 16 + 2 * tn + (j >> 4), a.n_tiles - 1);
    wptr[tn] = a.w + tile * k_tiles * 1024 + (16 * h + (j & 15)) * 16;
    wsptr[tn] = a.ws + tile * k_groups * 64 + 16 * h + (j & 15);
  }
  struct WStep {
    u32x4 w[TN][KK];
    uint32_t s[TN][2];      // of the 512 k that the step lies in
  };
  auto load_w = [&](int s, WStep& d) {
    const int kt = min(s_begin + s, steps - 1) * KT;
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        d.w[tn][kk] = *reinterpret_cast<const u32x4*>(wptr[tn] + static_cast<int64_t>(kt) * 1024 + kk * 512);
#pragma unroll
      for (int half = 0; half < 2; ++half) d.s[tn][half] = wsptr[tn][(kt >> 2) * 64 + half * 32];
    }
  };
  const uint8_t* xptr[XH];
  int park_at[XH];
#pragma unroll
  for (int p = 0; p < XH; ++p) {
    const int row = (p * kThreads + tid) >> 3, c = tid & 7;
    xptr[p] = a.x + static_cast<int64_t>(min(m0 + row, a.M - 1)) * a.ldx + c * 16;
    park_at[p] = row * 128 + (c ^ (row & 7)) * 16;
  }
  const uint8_t* xsptr[XS];
#pragma unroll
  for (int p = 0; p < XS; ++p) xsptr[p] = a.xs + static_cast<int64_t>(min(m0 + min(p * kThreads + tid, kRows - 1), a.M - 1)) * a.ldxs;
  struct XStep {
    u32x4 x[XH];
    uint32_t s[XS][KT];
  };
  auto load_x = [&](int s, XStep& d) {
    const int64_t at = min(s_begin + s, steps - 1);
#pragma unroll
    for (int p = 0; p < XH; ++p) d.x[p] = *reinterpret_cast<const u32x4*>(xptr[p] + at * 128);
#pragma unroll
    for (int p = 0; p < XS; ++p)
#pragma unroll
      for (int q = 0; q < KT; ++q) d.s[p][q] = *reinterpret_cast<const uint32_t*>(xsptr[p] + at * 4 * KT + 4 * q);
  };
  auto park_x = [&](int stage, const XStep& d) {
    unsigned char* to = lds + stage * kStage;
#pragma unroll
    for (int p = 0; p < XH; ++p) *reinterpret_cast<u32x4*>(to + park_at[p]) = d.x[p];
#pragma unroll
    for (int p = 0; p < XS; ++p)
      if (p * kThreads + tid < kRows) {
#pragma unroll
        for (int q = 0; q < KT; ++q) *reinterpret_cast<uint32_t*>(to + kRows * 128 + (q * kRows + p * kThreads + tid) * 4) = d.s[p][q];
      }
  };

  mx_f32x16 acc[MT][TN];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][tn][r] = 0.f;
  const int row_at = (wr * 32 * MT + j);
  auto multiply = [&](int s, int stage, const WStep& d) {
    const unsigned char* from = lds + stage * kStage;
    const int kt = (s_begin + s) * KT;
    uint32_t xs[MT][KT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int q = 0; q < KT; ++q)
        xs[t][q] = *reinterpret_cast<const uint32_t*>(from + kRows * 128 + (q * kRows + row_at + 32 * t) * 4) >> (8 * h);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      int wscale[TN];
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) wscale[tn] = static_cast<int>(d.s[tn][kk & 1] >> (8 * ((kt + kk / 2) & 3)));
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const unsigned char* row = from + (row_at + 32 * t) * 128;
        mx_i32x8 xo;
        if constexpr (BITS == kMx8)
          xo = mx_operand8(*reinterpret_cast<const u32x4*>(row + ((4 * kk + h) ^ (j & 7)) * 16),
                           *reinterpret_cast<const u32x4*>(row + ((4 * kk + 2 + h) ^ (j & 7)) * 16));
        else
          xo = mx_operand4(*reinterpret_cast<const u32x4*>(row + ((2 * kk + h) ^ (j & 7)) * 16));
        const int xscale = static_cast<int>(xs[t][kk / 2]);
#pragma unroll
        for (int tn = 0; tn < TN; ++tn) {
          if ((kk & 1) == 0)
            acc[t][tn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand4(d.w[tn][kk]), xo, acc[t][tn], 4, BITS == kMx8 ? 0 : 4, 0,
                                                                         wscale[tn], 0, xscale);
          else
            acc[t][tn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand4(d.w[tn][kk]), xo, acc[t][tn], 4, BITS == kMx8 ? 0 : 4, 0,
                                                                         wscale[tn], 2, xscale);
        }
      }
    }
  };

  WStep wring[PD];
  XStep xnext;
  load_x(0, xnext);
#pragma unroll
  for (int u = 0; u < PD; ++u) load_w(u, wring[u]);
  park_x(0, xnext);
  load_x(1, xnext);
  __syncthreads();
  for (int s0 = 0; s0 < n_steps; s0 += PD) {
#pragma unroll
    for (int u = 0; u < PD; ++u) {
      const int s = s0 + u;
      if (s < n_steps) {                          // the same in the whole workgroup
        park_x((u + 1) & 1, xnext);               // everybody is past the step that read that stage
        load_x(s + 2, xnext);
        multiply(s, u & 1, wring[u]);
        load_w(s + PD, wring[u]);
        __syncthreads();
      }
    }
  }

  // acc[t][tn][r] = C[m0 + 32 (MT wr + t) + j][n0 + 32 tn + 8 (r / 4) + 4 h + r % 4]
  if constexpr (kGate) {
    constexpr int kBits = EPI == kMxGate8 ? kMx8 : kMx4;
    if (n0 / 16 >= a.n_tiles) return;             // (whole blocks: the columns are a multiple of 512)
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float4 v[TN][2];
      uint32_t most = 0;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          v[tn][q] = float4{mx_silu_mul(acc[t][tn][4 * q], acc[t][tn][4 * q + 8]), mx_silu_mul(acc[t][tn][4 * q + 1], acc[t][tn][4 * q + 9]),
                            mx_silu_mul(acc[t][tn][4 * q + 2], acc[t][tn][4 * q + 10]), mx_silu_mul(acc[t][tn][4 * q + 3], acc[t][tn][4 * q + 11])};
          most = max(most, mx_max4(v[tn][q]));
        }
      const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
      const uint32_t code = mx_code<kBits>(max(both[0], both[1]));
      const int row = m0 + 32 * (MT * wr + t) + j;
      if (row < a.M) {
        uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.ldo;
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
          for (int q = 0; q < 2; ++q) mx_store4<kBits>(o, n0 / 2 + 16 * tn + 8 * q + 4 * h, mx_pack4<kBits>(v[tn][q], code));
        if (h == 0) a.out_scales[row * a.ldos + n0 / 64] = static_cast<uint8_t>(code);
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mx_store_sums<EPI>(a, blockIdx.y, m0 + 32 * (MT * wr + t) + j, n0 + 32 * tn + 8 * q + 4 * h,
                             mx_f32x4{acc[t][tn][4 * q], acc[t][tn][4 * q + 1], acc[t][tn][4 * q + 2], acc[t][tn][4 * q + 3]});
  }
}

// ---- launches

template <int BITS, int EPI, int RT, int CT, int WAVES, int U>
int mx_rows_launch(const MxArgs& a, int splits, hipStream_t s) {
  mx_gemm_rows_kernel<BITS, RT, CT, WAVES, U, EPI><<<dim3((a.n_tiles + CT - 1) / CT, splits), WAVES * kWave, 0, s>>>(a);
  return launch_status();
}

template <int BITS, int EPI, int MT, int TN, int RW, int CW, int PD>
int mx_tiles_launch(MxArgs a, int splits, hipStream_t s) {
  static OnceADevice asked;
  constexpr int kRows = 32 * MT * RW;
  constexpr size_t kLds = 2 * kRows * (128 + (BITS == kMx8 ? 4 : 8));
  const auto kernel = mx_gemm_tiles_kernel<BITS, MT, TN, RW, CW, PD, EPI>;
  if (const int e = ask_lds(asked, kLds, {reinterpret_cast<const void*>(kernel)})) return e;
  a.m_blocks = (a.M + kRows - 1) / kRows;
  a.n_blocks = (a.n_tiles + 2 * TN * CW - 1) / (2 * TN * CW);
  const int per_xcd = (a.m_blocks * a.n_blocks + 7) / 8;
  kernel<<<dim3(8 * per_xcd, splits), RW * CW * kWave, kLds, s>>>(a);
  return launch_status();
}

template <int BITS, int EPI>
int mx_launch(int variant, const MxArgs& a, int splits, hipStream_t s) {
  constexpr bool kGate = EPI == kMxGate8 || EPI == kMxGate4;
  switch (variant) {
    case 0: return mx_rows_launch<BITS, EPI, 1, kGate ? 4 : 2, 8, 2>(a, splits, s);
    case 1: return mx_rows_launch<BITS, EPI, 2, kGate ? 4 : 2, 8, 1>(a, splits, s);
    case 2: return mx_rows_launch<BITS, EPI, 4, kGate ? 4 : 2, 4, 1>(a, splits, s);
    case 3: return mx_tiles_launch<BITS, EPI, 1, 2, 2, 2, 2>(a, splits, s);
    case 4: return mx_tiles_launch<BITS, EPI, 2, 2, 2, 2, 2>(a, splits, s);
    case 5: return mx_tiles_launch<BITS, EPI, 4, 2, 1, 4, 2>(a, splits, s);
    case 6: return mx_tiles_launch<BITS, EPI, 4, 2, 2, 4, 2>(a, splits, s);
  }
  return static_cast<int>(hipErrorInvalidValue);
}

}  // namespace arle

using namespace arle;

extern "C" int arle_mx_gemm(int bits, int epilogue, int variant, const void* x, long long ldx, const void* xs, long long ldxs, const void* w,
                            const void* ws, void* out, long long ldo, long long split_stride, void* out_scales, long long ldos, int M, int N,
                            int n_tiles, int k_tiles, int splits, int per_split, int vec, void* stream) {
  const MxArgs a = {static_cast<const uint8_t*>(x), ldx, static_cast<const uint8_t*>(xs), ldxs, static_cast<const uint8_t*>(w),
                    static_cast<const uint32_t*>(ws), out, ldo, split_stride, static_cast<uint8_t*>(out_scales), ldos, M, N, n_tiles, k_tiles,
                    per_split, vec, 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto with = [&](auto b) {
    constexpr int kBits = decltype(b)::value;
    switch (epilogue) {
      case kMxF32: return mx_launch<kBits, kMxF32>(variant, a, splits, s);
      case kMxBf16: return mx_launch<kBits, kMxBf16>(variant, a, splits, s);
      case kMxGate8: return mx_launch<kBits, kMxGate8>(variant, a, splits, s);
      case kMxGate4: return mx_launch<kBits, kMxGate4>(variant, a, splits, s);
    }
    return static_cast<int>(hipErrorInvalidValue);
  };
  return bits == kMx8 ? with(std::integral_constant<int, kMx8>{}) : with(std::integral_constant<int, kMx4>{});
}
