// Windowed prefill attention for the shapes that the pair kernel (paged_prefill.hip) does not take:
// head dims 32, 64 and 256, and at 128 pages of fewer than 16 keys and a scale that is not positive;
// any GQA group, 16-bit queries over a pool of their type or fp8. A query at position p sees the keys
// j <= p with j > p - window or j < sinks.
//
// Design:
//  * a work item is kRows rows of one (sequence, kv head), a row being one (query position, query
//    head of the group) pair, the group's heads of a position next to each other: every head of the
//    group shares the staged K and V whatever the group, and a chunk of a few tokens fills its
//    rows with its heads.
//  * an item walks the entries of its key list (paged_attention.hpp): exactly the sinks and the
//    keys from its first query's window to its last query, 64 a tile.
//  * 4 waves of 32 rows (two blocks of 16, one K / V fragment read from LDS feeding the MFMAs of
//    both), at D = 256 8 waves of 16, K and V row-major in LDS. S^T = K Q^T on v_mfma_f32_16x16x32:
//    a lane holds one row's scores of keys 4 g + i of every 16 (g = lane / 16). The PV product sums
//    over keys, so P^T is used as the scores lie: of a step of 32 keys a lane has 4 g .. 4 g + 3 and
//    16 + 4 g .. + 3, and V is read transposed (ds_read_b64_tr_b16) in that order.
//  * LDS chunks are swizzled by their row so that the rows that one read serves lie in distinct banks.
//  * the next tile's rows are requested before a tile is computed and stored to LDS after it, into a
//    second buffer; page ids one tile before that.
//  * online softmax in float32 in log2 units against the exact running maximum, so that a row's
//    largest weight is 1 and not rounded; the weights are rounded to the queries' type for the MFMA,
//    their sum is not.
//
// What bounds it: LDS reads. A wave reads a tile's K and V, 256 D bytes, for 2 x 64 x D x 16 kBlocks
// multiply-adds: with 32 rows as many cycles of the CU's LDS as of its four matrix cores, with
// 16 twice as many; and with few workgroups the wait for the next tile. Head dim 256, 8 query heads
// over 2: chunks of 54 and 163 tokens with a window of 1007 62 us, 601 and 1805 over fp8 with 380 36
// (the register-staged causal kernel, given windows, spilled there: 170 and 84). At 256, 4 waves of
// 32 rows, one a SIMD: 111 and 53. At 128 the pair kernel's waves are ahead where they serve: one
// head a kv head, two chunks of 520-1562 tokens with 518, 27 us against 39.

#include <climits>
#include <type_traits>

#include "common.hpp"
#include "paged_attention.hpp"
#include "window_list.hpp"

namespace mvllm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;     // keys

template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  __device__ static f32x4 run(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <> struct Mma16<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  __device__ static f32x4 run(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack2(float lo, float hi) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
};

// Eight consecutive pool elements as loaded, and as the eight 16-bit elements the MFMAs read.
template <typename TQ, typename TKV> struct Raw {
  u32x4 w;
  __device__ void load(const char* p) { w = load16(p); }
  __device__ u32x4 elements(float) const { return w; }
};
template <typename TQ> struct Raw<TQ, fp8_t> {
  u32x2 w;
  __device__ void load(const char* p) { w = *reinterpret_cast<const u32x2*>(p); }
  __device__ u32x4 elements(float scale) const {
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
      out[2 * i] = Mma16<TQ>::pack2(lo[0] * scale, lo[1] * scale);
      out[2 * i + 1] = Mma16<TQ>::pack2(hi[0] * scale, hi[1] * scale);
    }
    return out;
  }
};

// kBlocks: 16-row blocks of a wave.
template <typename TQ, typename TKV, int D, int kWaves, int kBlocks>
__global__ __launch_bounds__(kWaves * kWave, 2) void window_prefill_kernel(const PagedParams p) {
  constexpr bool kFp8 = std::is_same_v<TKV, fp8_t>;
  constexpr int kThreads = kWaves * kWave;
  constexpr int kRows = 16 * kWaves * kBlocks;
  constexpr int kChunks = D / 8;                     // 16-byte chunks of a staged row
  constexpr int kUnits = kTile * kChunks / kThreads;  // chunks of K (and of V) a thread stages
  constexpr int kRowBytes = 2 * D;
  constexpr int kRowsPerLine = kRowBytes < 256 ? 256 / kRowBytes : 1;  // rows side by side in the banks
  constexpr int kPairs = kChunks / 2;
  constexpr int kKMask = (kChunks < 16 ? kChunks : 16) - 1, kVMask = (kPairs < 8 ? kPairs : 8) - 1;
  constexpr int kSteps = D / 32, kDims = D / 16;
  __shared__ __align__(1024) char k_lds[2][kTile * kRowBytes];
  __shared__ __align__(1024) char v_lds[2][kTile * kRowBytes];

  const int seq = blockIdx.y, kvh = blockIdx.x;
  const int len = sload(p.seq_lens + seq);
  if (len < p.pf_min_len) return;  // a decode row: the decode kernel has it
  const int held = sload(p.context_lens + seq);
  const int group = p.hq / p.hk;
  const int rows = len * group;
  // The items of a sequence's last queries first, which see the most keys.
  const int item = (rows + kRows - 1) / kRows - 1 - static_cast<int>(blockIdx.z);
  if (item < 0) return;
  const int row0 = item * kRows, row_end = min(row0 + kRows, rows);
  const int q_row0 = sload(p.cu_seqlens_q + seq);
  const int offset = held - len;
  const WindowList list = window_list<1>(p, offset + row0 / group);
  const int keys = offset + (row_end - 1) / group + 1 - list.gap;  // entries the item walks
  const int tiles = (keys + kTile - 1) / kTile;

  const int tid = threadIdx.x, lane = tid % kWave;
  if (tiles <= 0) {  // no key at all: zeros
    for (int i = tid; i < (row_end - row0) * (D / 2); i += kThreads) {
      const int row = row0 + i / (D / 2), at = row / group;
      const int64_t head = static_cast<int64_t>(q_row0 + at) * p.hq + kvh * group + (row - at * group);
      static_cast<uint32_t*>(p.out)[head * (D / 2) + i % (D / 2)] = 0;
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n16 = lane & 15, g = lane >> 4;

  // ---- this wave's rows.
  const int w_row0 = row0 + wave * 16 * kBlocks;
  const bool w_active = w_row0 < row_end;
  const int w_last = min(w_row0 + 16 * kBlocks, row_end) - 1;
  const int w_full = offset + w_row0 / group + 1 - list.gap;          // entries all its rows see
  const int w_end = w_active ? offset + w_last / group + 1 - list.gap : 0;
  int visible[kBlocks];
  u32x4 qop[kBlocks][kSteps];
  const float raw_c = p.scale * kLog2e;
  const float score_c = fmaxf(fabsf(raw_c), 1e-30f);  // (a negative scale's sign is moved into Q)
  const uint32_t q_sign = raw_c < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int row = min(w_row0 + 16 * b + n16, row_end - 1);
    const int at = row / group;
    visible[b] = w_row0 + 16 * b + n16 < row_end ? offset + at + 1 - list.gap : INT_MIN;
    const char* src = static_cast<const char*>(p.q) +
                      ((static_cast<int64_t>(q_row0 + at) * p.hq + kvh * group + (row - at * group)) * D + 8 * g) * 2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qop[b][s] = load16(src + 64 * s) ^ q_sign;
  }
  f32x4 o[kBlocks][kDims];
  float m_run[kBlocks], l_run[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m_run[b] = -INFINITY;
    l_run[b] = 0.0f;
  }

  // ---- staging: unit u of a thread is chunk tid % kChunks of key (tid + 256 u) / kChunks.
  const char* kpool = static_cast<const char*>(p.k_pool);
  const char* vpool = static_cast<const char*>(p.v_pool);
  const int32_t* table = p.block_tables + static_cast<int64_t>(seq) * p.max_blocks;
  const int last = held - list.gap - 1;
  const uint32_t in_row = static_cast<uint32_t>(kvh * p.kv_head_bytes) + tid % kChunks * 8 * Elem<TKV>::kBytes;
  auto entry = [&](int t, int u) __attribute__((always_inline)) {
    return list_position(list, min(t * kTile + (tid + u * kThreads) / kChunks, last));
  };
  int page[kUnits];
  Raw<TQ, TKV> kr[kUnits], vr[kUnits];
  float ks[kUnits], vs[kUnits];
  auto fetch_pages = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) page[u] = table[entry(t, u) >> p.block_shift];
  };
  auto load_tile = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int id = held_page(p, page[u]);
      const int64_t slot = (static_cast<int64_t>(id) << p.block_shift) + (entry(t, u) & p.block_mask);
      const int64_t at = slot * p.kv_row_bytes + in_row;
      kr[u].load(kpool + at);
      vr[u].load(vpool + at);
      ks[u] = kFp8 ? p.k_scales[static_cast<int64_t>(id) * p.hk + kvh] : 1.0f;
      vs[u] = kFp8 ? p.v_scales[static_cast<int64_t>(id) * p.hk + kvh] : 1.0f;
    }
  };
  auto store_tile = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int key = (tid + u * kThreads) / kChunks, chunk = tid % kChunks, line = key / kRowsPerLine;
      *reinterpret_cast<u32x4*>(&k_lds[buf][key * kRowBytes + (chunk ^ (line & kKMask)) * 16]) = kr[u].elements(ks[u]);
      *reinterpret_cast<u32x4*>(
          &v_lds[buf][key * kRowBytes + (((chunk >> 1) ^ (line & kVMask)) * 2 + (chunk & 1)) * 16]) =
          vr[u].elements(vs[u]);
    }
  };

  auto compute = [&](int t, int buf) __attribute__((always_inline)) {
    const int key0 = t * kTile;
    if (!w_active || key0 >= w_end) return;
    f32x4 s[kBlocks][4];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) s[b][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const int key = 16 * kb + n16, line = key / kRowsPerLine;
        const u32x4 a = *reinterpret_cast<const u32x4*>(
            &k_lds[buf][key * kRowBytes + ((4 * st + g) ^ (line & kKMask)) * 16]);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) s[b][kb] = Mma16<TQ>::run(a, qop[b][st], s[b][kb]);
      }
    }
    if (key0 + kTile > w_full || (key0 < w_end - p.window && key0 + kTile > p.sinks)) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int hi = visible[b] == INT_MIN ? INT_MIN : visible[b] - key0 - 4 * g;
        const int lo = visible[b] == INT_MIN ? INT_MIN : visible[b] - p.window - key0 - 4 * g;
        const int front = p.sinks - key0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = 16 * kb + i;
            if (e >= hi || (e >= front && e < lo)) s[b][kb][i] = -INFINITY;
          }
        }
      }
    }
    u32x4 pop[kBlocks][2];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      float most = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, s[b][kb][i]);
      }
      most = fmaxf(most, __shfl_xor(most, 16, kWave));
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      const float m_new = fmaxf(m_run[b], most * score_c);
      if (__builtin_amdgcn_ballot_w64(m_new > m_run[b]) != 0) {
        const float alpha = m_new == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[b] - m_new);
        m_run[b] = m_new;
        l_run[b] *= alpha;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[b][d] *= alpha;
      }
      const float neg_mu = m_run[b] == -INFINITY ? 0.0f : -m_run[b];
      float sum = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = __builtin_amdgcn_exp2f(fmaf(s[b][2 * h + i / 4][i % 4], score_c, neg_mu));
          sum += w[i];
        }
        pop[b][h] = u32x4{Mma16<TQ>::pack2(w[0], w[1]), Mma16<TQ>::pack2(w[2], w[3]),
                          Mma16<TQ>::pack2(w[4], w[5]), Mma16<TQ>::pack2(w[6], w[7])};
      }
      l_run[b] += sum;
    }
    // O^T += V^T P^T. Lane L of a 16-lane group reads four dims of one key (L / 4) and gets dim L of
    // the group's four keys.
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
    const uint32_t base = lds_address(v_lds[buf]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        u32x4 a;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = 32 * h + 16 * half + 4 * g + n16 / 4, line = key / kRowsPerLine;
          const uint32_t at = base + key * kRowBytes + (d ^ (line & kVMask)) * 32 + (n16 & 3) * 8;
          const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              reinterpret_cast<lds_v4i16*>(at)));
          a[2 * half] = v[0];
          a[2 * half + 1] = v[1];
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) o[b][d] = Mma16<TQ>::run(a, pop[b][h], o[b][d]);
      }
    }
  };

  fetch_pages(0);
  load_tile(0);
  if (tiles > 1) fetch_pages(1);
  store_tile(0);
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
    const bool more = t + 1 < tiles;
    if (more) load_tile(t + 1);
    if (t + 2 < tiles) fetch_pages(t + 2);
    __builtin_amdgcn_sched_barrier(0);
    compute(t, t % 2);
    __builtin_amdgcn_sched_barrier(0);
    if (more) store_tile((t + 1) % 2);
    __syncthreads();
  }

#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    float l = l_run[b];
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    const int row = w_row0 + 16 * b + n16;
    if (row >= row_end) continue;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int at = row / group;
    char* dst = static_cast<char*>(p.out) +
                ((static_cast<int64_t>(q_row0 + at) * p.hq + kvh * group + (row - at * group)) * D + 4 * g) * 2;
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      *reinterpret_cast<u32x2*>(dst + 32 * d) =
          u32x2{Mma16<TQ>::pack2(o[b][d][0] * inv, o[b][d][1] * inv),
                Mma16<TQ>::pack2(o[b][d][2] * inv, o[b][d][3] * inv)};
    }
  }
}

template <typename TQ, typename TKV, int D, int kWaves, int kBlocks>
hipError_t launch(const PagedParams& p, int max_query_len, hipStream_t stream) {
  constexpr int kRows = 16 * kWaves * kBlocks;
  const int64_t rows = static_cast<int64_t>(max_query_len) * (p.hq / p.hk);
  const int64_t items = (rows + kRows - 1) / kRows;
  if (rows >= INT_MAX || items > 65535 || p.num_seqs > 65535) return hipErrorInvalidValue;
  window_prefill_kernel<TQ, TKV, D, kWaves, kBlocks>
      <<<dim3(p.hk, p.num_seqs, static_cast<unsigned>(items)), kWaves * kWave, 0, stream>>>(p);
  return hipGetLastError();
}

template <typename TQ, typename TKV>
hipError_t launch_t(const PagedParams& p, int head_dim, int max_query_len, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch<TQ, TKV, 32, 4, 2>(p, max_query_len, stream);
    case 64: return launch<TQ, TKV, 64, 4, 2>(p, max_query_len, stream);
    case 128: return launch<TQ, TKV, 128, 4, 2>(p, max_query_len, stream);
    case 256: return launch<TQ, TKV, 256, 8, 1>(p, max_query_len, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

bool window_prefill_supported(int q_dtype, int kv_dtype, int head_dim) {
  return (q_dtype == kBF16 || q_dtype == kF16) && (kv_dtype == q_dtype || kv_dtype == kFP8E4M3) &&
         (head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256);
}

hipError_t launch_window_prefill(const PagedParams& p, int q_dtype, int kv_dtype, int head_dim,
                                 int max_query_len, hipStream_t stream) {
  const bool fp8 = kv_dtype == kFP8E4M3;
  if (q_dtype == kBF16) {
    return fp8 ? launch_t<bf16_t, fp8_t>(p, head_dim, max_query_len, stream)
               : launch_t<bf16_t, bf16_t>(p, head_dim, max_query_len, stream);
  }
  if (q_dtype == kF16) {
    return fp8 ? launch_t<f16_t, fp8_t>(p, head_dim, max_query_len, stream)
               : launch_t<f16_t, f16_t>(p, head_dim, max_query_len, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mvllm
