// Attention of few query rows over the paged 8-bit KV cache: one pass over the codes with
// m16n8k16 tensor-core products on fp16 operands.
//
// Codes convert to fp16 exactly (e4m3 by the hardware conversion, int8 through the integers
// 1024 + u that fp16 represents), queries are multiplied by a power of two that puts each row's
// largest element in [2^14, 2^15), so the scores carry the inputs' own precision; probabilities
// round to fp16 (2^-11).  ks_j multiplies scores, vs_j probabilities, relative to the largest
// vs of the warp so far (O is rescaled when it grows, as when the row maximum does).
//
// Operands come straight from global memory into registers; neither product needs a byte moved
// between lanes, because a contraction may run over its index in any order:
//   S = Q K^T: lane (g, t) loads 16 consecutive bytes of key 8n + g at channel 64h + 16t; bytes
//     4s .. 4s + 3 are its B fragment of step (h, s), the query fragments are laid out alike;
//   O^T = V^T P^T: lane (g, t) loads 16 channels at 16g of keys 2t, 2t + 1, 2t + 8, 2t + 9 of a
//     16-key group; byte permutes pair two keys of one channel, and m-tile i takes channels
//     16g + 2i (rows 0-7) and 16g + 2i + 1 (rows 8-15).  S's accumulators are P^T's B fragment.
// With the queries as the 8 columns of O^T, up to 8 rows cost one product a group and 32
// accumulators (RT = 1); 9 to 16 rows two (RT = 2).
//
// What bounds it: HBM.  A warp reads 32 keys (8 KB) at a time; the next 32 keys' loads are issued
// as soon as the registers are free, page ids one block earlier still.
#include <algorithm>
#include <type_traits>

#include "kv_attention.cuh"
#include "sm100.cuh"

namespace ntb {
namespace kv {
namespace {

constexpr int kThreads = 128;
constexpr int kUnit = 128;            // keys of a unit: 32 a warp
constexpr float kGrow = 6.f;          // rows rescale when their maximum grows by more (p <= 2^6)

// Four codes -> two fp16 pairs (bytes 0, 1 and 2, 3).
template <int CODE>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == NTB_F8E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // w holds code + 128 in each byte: 0x6400 | u is the fp16 number 1024 + u
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 k = __floats2half2_rn(1152.f, 1152.f);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), k);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), k);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
template <int CODE>
__device__ __forceinline__ uint32_t bias(uint32_t w) {
  return CODE == NTB_I8 ? w ^ 0x80808080u : w;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Codes are read once: no L1 allocation.
template <int W>
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&r)[W]) {
  if constexpr (W == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
}

template <int D, int RT>
constexpr int min_blocks() {
  return D == 128 ? (RT == 1 ? 3 : 2) : (RT == 1 ? 5 : 4);
}

template <typename T, int CODE, int D, int RT>
__global__ void __launch_bounds__(kThreads, min_blocks<D, RT>()) decode_kernel(AttnArgs a, int t_shift, int q_vec) {
  constexpr int H64 = D / 64;       // 16-byte loads of a key row per lane
  constexpr int VW = D / 32;        // words of a lane's V channels: 4 (D 128) or 2 (D 64)
  constexpr int MT = D / 16;        // m-tiles of O^T
  constexpr int ROWS = 8 * RT;
  constexpr int OS = D + 4;         // padded row of the merge buffer
  extern __shared__ int pre[];
  __shared__ __align__(16) float so[4][ROWS][OS];
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  grid_dependency_launch();  // the joining kernel may start; it waits for this one before it reads
  prefix_units<kThreads>(a, pre);
  const Line line(a, pre);
  if ((int)blockIdx.x >= line.blocks) return;
  const int64_t lo = line.begin(blockIdx.x), hi = line.begin(blockIdx.x + 1);

  for (int64_t pos = lo; pos < hi;) {
    const Piece pc = piece_at(a, line, pre, pos, lo, hi);
    pos = pc.next;
    const int len = row_length(a, pc.b), start = row_start(a, pc.b, len);
    const int r0 = pc.tile * ROWS;
    // ------------------------------------------------------------------- queries ----
    uint32_t qa[RT][H64 * 4][2];
    float rowsc[RT];  // scores of this lane's row(s): accumulator -> base-2 logits, without ks
    int kmax[RT];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const int r = r0 + g + 8 * x;
      float v[H64][16];
      kmax[x] = r < a.rows ? last_key(a, len, start, r / a.group) : -1;
      if (r < a.rows) {
        const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)pc.b * a.q_b +
                      (int64_t)(pc.head * a.group + r % a.group) * a.q_h + (int64_t)(r / a.group) * a.q_s + 16 * t;
#pragma unroll
        for (int h = 0; h < H64; ++h) {
          if (q_vec) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const ew::Vec<T, 8> w = *reinterpret_cast<const ew::Vec<T, 8>*>(qp + 64 * h + 8 * e);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[h][8 * e + i] = cvt<float>(w.v[i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[h][i] = cvt<float>(qp[64 * h + i]);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < H64; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) v[h][i] = 0.f;
      }
      float amax = 0.f;
#pragma unroll
      for (int h = 0; h < H64; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[h][i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int be = (int)(__float_as_uint(amax) >> 23);
      const int e = be == 255 ? 0 : min(max(141 - be, -110), 110);  // amax * 2^e in [2^14, 2^15)
      const float up = pow2(e);
      rowsc[x] = a.scale * kLog2eF * pow2(-e);
#pragma unroll
      for (int h = 0; h < H64; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          qa[x][h * 4 + s][0] = pack_f16(v[h][4 * s] * up, v[h][4 * s + 1] * up);
          qa[x][h * 4 + s][1] = pack_f16(v[h][4 * s + 2] * up, v[h][4 * s + 3] * up);
        }
    }
    // every row of the tile sees the keys up to k_low; none sees a key at or past k_end
    const int k_low = last_key(a, len, start, r0 / a.group);
    const int k_end = min(len, last_key(a, len, start, (min(r0 + ROWS, a.rows) - 1) / a.group) + 1);

    float m[RT], l[RT], vref = 1.17549435e-38f, inv_vref = 1.f / vref;
    float o[RT][MT][4];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;
    }
    const uint8_t* kbase = a.c.key + (int64_t)pc.head * a.c.k_h + (int64_t)g * a.c.k_t + 16 * t;
    const uint8_t* vbase = a.c.value + (int64_t)pc.head * a.c.v_h + (int64_t)(2 * t) * a.c.v_t + 4 * VW * g;
    const float* ksb = a.c.key_scale + (int64_t)pc.head * a.c.ks_h;
    const float* vsb = a.c.value_scale + (int64_t)pc.head * a.c.vs_h;

    // ---------------------------------------------------- loads of one block of 32 keys ----
    auto load_ids = [&](int u, int (&id)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = u * kUnit + warp * 32 + 16 * j;
        id[j] = -1;
        if (u < pc.u1 && key < k_end)
          id[j] = page_of(a.table, a.c.P, pc.b, t_shift >= 0 ? key >> t_shift : key / a.c.T);
      }
    };
    auto in_page = [&](int key) { return t_shift >= 0 ? key & (a.c.T - 1) : key % a.c.T; };
    uint32_t kr[4][H64][4], vr[2][4][VW];
    float ks[2], vs[2], vs_next[2];
    auto load_k = [&](int u, const int (&id)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int page = max(id[j], 0);  // a hole reads page 0 and is masked
        ks[j] = ksb[(int64_t)page * a.c.ks_p];
        vs_next[j] = id[j] < 0 ? 0.f : vsb[(int64_t)page * a.c.vs_p];
        const uint8_t* p = kbase + (int64_t)page * a.c.k_p +
                           (int64_t)in_page(u * kUnit + warp * 32 + 16 * j) * a.c.k_t;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < H64; ++h)
            load_codes<4>(p + (int64_t)n * 8 * a.c.k_t + 64 * h, kr[2 * j + n][h]);
      }
    };
    auto load_v = [&](int u, const int (&id)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* p = vbase + (int64_t)max(id[j], 0) * a.c.v_p +
                           (int64_t)in_page(u * kUnit + warp * 32 + 16 * j) * a.c.v_t;
#pragma unroll
        for (int k = 0; k < 4; ++k) load_codes<VW>(p + (int64_t)((k & 1) + 8 * (k >> 1)) * a.c.v_t, vr[j][k]);
      }
    };

    int id[2], id_next[2];
    auto any_key = [&](int u) { return u < pc.u1 && u * kUnit + warp * 32 < k_end; };
    load_ids(pc.u0, id);
    if (any_key(pc.u0)) {
      load_k(pc.u0, id);
      load_v(pc.u0, id);
    }
    load_ids(pc.u0 + 1, id_next);
    for (int u = pc.u0; u < pc.u1; ++u) {
      const int kw = u * kUnit + warp * 32;
      if (kw >= k_end) break;  // (later blocks too)
      // ------------------------------------------------------------- S = Q K^T ----
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      // keys innermost: four independent accumulators in turn
#pragma unroll
      for (int h = 0; h < H64; ++h)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint32_t b0, b1;
            widen4<CODE>(bias<CODE>(kr[n][h][w]), b0, b1);
            mma_f16(s[n], qa[0][h * 4 + w][0], RT == 2 ? qa[RT - 1][h * 4 + w][0] : 0u, qa[0][h * 4 + w][1],
                    RT == 2 ? qa[RT - 1][h * 4 + w][1] : 0u, b0, b1);
          }
      const float ks_cur[2] = {ks[0], ks[1]};
      const bool hole[2] = {id[0] < 0, id[1] < 0};
      vs[0] = vs_next[0];
      vs[1] = vs_next[1];
      if (any_key(u + 1)) load_k(u + 1, id_next);
      // ------------------------------------------------------------- softmax ----
      const bool edge = kw + 31 > k_low || hole[0] || hole[1];
      float alpha[RT];
      bool grown = false;
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        float mb = -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float sc = rowsc[x] * ks_cur[n >> 1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = s[n][2 * x + e] * sc;
            if (edge) {
              const int key = kw + 8 * n + 2 * t + e;
              if (key > kmax[x] || hole[n >> 1]) v = -INFINITY;
            }
            s[n][2 * x + e] = v;
            mb = fmaxf(mb, v);
          }
        }
        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
        alpha[x] = 1.f;
        if (mb > m[x] + kGrow) {
          alpha[x] = exp2f(m[x] - mb);  // 0 at the first block that the row sees
          m[x] = mb;
          grown = true;
        }
      }
      float vmul = 1.f;
      const float vtop = fmaxf(fabsf(vs[0]), fabsf(vs[1]));
      if (vtop > vref) {  // the same for every lane
        vmul = vref / vtop;
        vref = vtop;
        inv_vref = 1.f / vtop;
      }
      if (__any_sync(0xffffffffu, grown) || vmul != 1.f) {
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          l[x] *= alpha[x];
          // O^T's columns are rows 2t and 2t + 1, whose statistics lanes 8t and 8t + 4 hold
          const float a0 = __shfl_sync(0xffffffffu, alpha[x], 8 * t) * vmul;
          const float a1 = __shfl_sync(0xffffffffu, alpha[x], 8 * t + 4) * vmul;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[x][i][0] *= a0;
            o[x][i][1] *= a1;
            o[x][i][2] *= a0;
            o[x][i][3] *= a1;
          }
        }
      }
      uint32_t pb[RT][2][2];
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        const float ref = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float p0 = sm100::ex2_approx(s[n][2 * x] - ref), p1 = sm100::ex2_approx(s[n][2 * x + 1] - ref);
          l[x] += p0 + p1;
          const float f = vs[n >> 1] * inv_vref;
          pb[x][n >> 1][n & 1] = pack_f16(p0 * f, p1 * f);
        }
      }
      // codes past the last key and in page 0 for a hole hold anything: 0 * NaN would not be 0
      if (kw + 32 > k_end || hole[0] || hole[1]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (hole[j] || kw + 16 * j + 2 * t + (k & 1) + 8 * (k >> 1) >= k_end)
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[j][k][w] = 0u;
      }
      // ------------------------------------------------------------- O^T += V^T P^T ----
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t v0 = bias<CODE>(vr[j][0][w]), v1 = bias<CODE>(vr[j][1][w]);
          const uint32_t v2 = bias<CODE>(vr[j][2][w]), v3 = bias<CODE>(vr[j][3][w]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x01 = __byte_perm(v0, v1, i ? 0x7362 : 0x5140);
            const uint32_t x23 = __byte_perm(v2, v3, i ? 0x7362 : 0x5140);
            uint32_t a0, a1, a2, a3;
            widen4<CODE>(x01, a0, a1);
            widen4<CODE>(x23, a2, a3);
#pragma unroll
            for (int x = 0; x < RT; ++x) mma_f16(o[x][2 * w + i], a0, a1, a2, a3, pb[x][j][0], pb[x][j][1]);
          }
        }
      if (any_key(u + 1)) load_v(u + 1, id_next);
      id[0] = id_next[0];
      id[1] = id_next[1];
      load_ids(u + 2, id_next);
    }
    // --------------------------------------------------- join the four warps' results ----
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (t == 0) {
        sm_m[warp][8 * x + g] = m[x];
        sm_l[warp][8 * x + g] = l[x];
      }
      // channels 4 VW g + 2i (elements 0, 1) and + 2i + 1 (2, 3) of rows 2t and 2t + 1
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < MT; i += 2)
          *reinterpret_cast<float4*>(&so[warp][8 * x + 2 * t + e][4 * VW * g + 2 * i]) =
              make_float4(o[x][i][e] * vref, o[x][i][2 + e] * vref, o[x][i + 1][e] * vref, o[x][i + 1][2 + e] * vref);
    }
    __syncthreads();
    const int rows = min(ROWS, a.rows - r0);
    for (int idx = threadIdx.x; idx < rows * D; idx += kThreads) {
      const int rt = idx / D, d = idx % D, r = r0 + rt;
      float M = sm_m[0][rt];
#pragma unroll
      for (int w = 1; w < 4; ++w) M = fmaxf(M, sm_m[w][rt]);
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2f(sm_m[w][rt] - ref);
        L = fmaf(sm_l[w][rt], f, L);
        acc = fmaf(so[w][rt][d], f, acc);
      }
      if (pc.whole) {
        reinterpret_cast<T*>(a.o)[(int64_t)pc.b * a.o_b + (int64_t)(pc.head * a.group + r % a.group) * a.o_h +
                                  (int64_t)(r / a.group) * a.o_s + d] = cvt<T>(L == 0.f ? 0.f : acc / L);
      } else {
        float* part = a.part + (int64_t)pc.slot * slot_floats(a.tile, D);
        part[rt * D + d] = acc;
        if (d == 0) {
          part[a.tile * D + 2 * rt] = M;
          part[a.tile * D + 2 * rt + 1] = L;
        }
      }
    }
    __syncthreads();  // before the next piece writes the merge buffers
  }
}

template <typename T, int CODE, int D, int RT>
int go(const AttnArgs& a, cudaStream_t st, int* blocks) {
  auto k = decode_kernel<T, CODE, D, RT>;
  if (blocks != nullptr) {  // asked for a full batch's unit counts, whatever this launch's batch
    *blocks = resident_blocks((const void*)k, kThreads, sizeof(int) * (a.nb + 1));
    return NTB_OK;
  }
  const bool pow2_page = (a.c.T & (a.c.T - 1)) == 0;
  int shift = 0;
  while (pow2_page && (1 << shift) < a.c.T) ++shift;
  const int q_vec = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && (a.q_b % 8 == 0 || a.table.B == 1) &&
                    (a.q_h % 8 == 0 || a.Hq == 1) && (a.q_s % 8 == 0 || a.Sq == 1);
  k<<<a.G, kThreads, sizeof(int) * (a.nb + 1), st>>>(a, pow2_page ? shift : -1, q_vec);
  NTB_LAUNCH_CHECK();
  return NTB_OK;
}

template <typename T, int CODE>
int go_d(const AttnArgs& a, cudaStream_t st, int* blocks) {
  if (a.c.D == 128) return a.tile == 8 ? go<T, CODE, 128, 1>(a, st, blocks) : go<T, CODE, 128, 2>(a, st, blocks);
  return a.tile == 8 ? go<T, CODE, 64, 1>(a, st, blocks) : go<T, CODE, 64, 2>(a, st, blocks);
}

int go_any(const AttnArgs& a, int dtype, cudaStream_t st, int* blocks) {
  if (dtype == NTB_BF16)
    return a.c.code == NTB_F8E4M3 ? go_d<__nv_bfloat16, NTB_F8E4M3>(a, st, blocks)
                                  : go_d<__nv_bfloat16, NTB_I8>(a, st, blocks);
  return a.c.code == NTB_F8E4M3 ? go_d<__half, NTB_F8E4M3>(a, st, blocks) : go_d<__half, NTB_I8>(a, st, blocks);
}

}  // namespace

// 16-bit queries, head_dim 64 or 128, pages that hold whole 16-key groups, 16-byte rows.
bool decode_takes(const AttnArgs& a, int dtype) {
  const Layer& c = a.c;
  auto al = [](const uint8_t* p, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % 16 == 0 && s1 % 16 == 0 && s2 % 16 == 0;
  };
  return (dtype == NTB_BF16 || dtype == NTB_F16) && (c.D == 64 || c.D == 128) && c.T % 16 == 0 && c.P > 0 &&
         al(c.key, c.k_p, c.k_h, c.k_t) && al(c.value, c.v_p, c.v_h, c.v_t);
}

int decode_plan(AttnArgs* a, int dtype) {
  a->tile = a->rows <= 8 ? 8 : 16;
  a->unit = kUnit;
  a->tiles = (a->rows + a->tile - 1) / a->tile;
  return go_any(*a, dtype, nullptr, &a->G);
}

int decode_launch(const AttnArgs& a, int dtype, cudaStream_t st) { return go_any(a, dtype, st, nullptr); }

}  // namespace kv
}  // namespace ntb
