// The rotating append: RoPE of q and k, and the write of k and v into the paged cache, in one
// launch. No counterpart in the reference, whose caller runs two ropes and PagedKvPool.write
// (model/qwen3_paged.py:76-80, block/kv_pool.py:116-155).
//
//   q_out[t] = rope(q[t]),  k_pool[slot[t]] = rope(k[t]),  v_pool[slot[t]] = v[t]
//   rope(x)  = x cos(p) + rotate_half(x) sin(p) at the token's position p: with the halves
//              (a, b) of a head vector, (a cos_lo - b sin_lo, b cos_hi + a sin_hi)
//
// Memory-bound: q is read and written, k and v read and written once, against 3 flops an
// element. A thread owns 8 elements of the lower half and the 8 they turn with, so the rotation
// needs no other lane, and for large calls does several heads of one token, whose position and
// cos / sin pieces (128 bytes a thread, against 32 of a head) it then loads once.
//
// A 16-bit or float32 pool of the inputs' type takes the rows as rope then a copy give them, bit for
// bit. An fp8 page keeps a power-of-two scale per kv head for K and for V, as kv_write.hip
// describes (grown as the page fills, its rows re-encoded when it grows); K is quantised from the
// float32 rotation, without a rounding to the inputs' type between. There a workgroup takes a window of
// tokens and one kv head, with the runs (tokens on consecutive rows of one page) that start in it: every
// thread a row's piece of K or of V, a run's two maxima meet in LDS, and each row is rotated, scaled
// and stored by the thread that loaded it. (One workgroup for a run's heads together, a thread walking
// the run's rows, as the plain write has it, would hold a page's rotated rows in float32, 256 registers
// a thread.)

#include <algorithm>

#include "common.hpp"
#include "paged_attention.hpp"
#include "rope_write.hpp"

namespace mvllm {

namespace {

constexpr int E = 8;  // elements of a piece

// Eight consecutive elements as they are stored: one 16-byte chunk, or two of float32.
template <typename T> struct Piece {
  static constexpr int kChunks = E / Chunk<T>::kN;
  u32x4 w[kChunks];
  __device__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) w[i] = nt_load16(p + 16 * i);
  }
  __device__ void store(char* p) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) store16(p + 16 * i, w[i]);
  }
  __device__ void unpack(float (&f)[E]) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) Chunk<T>::unpack(w[i], f + i * Chunk<T>::kN);
  }
  __device__ void pack(const float (&f)[E]) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) w[i] = pack_chunk<T>(f + i * Chunk<T>::kN);
  }
};

// A thread's pieces of one position's cos and sin rows. A position outside the tables turns every
// vector to NaN and reads nothing past them.
struct Angles {
  float cl[E], sl[E], ch[E], sh[E];
  __device__ void load(const RopeWriteParams& p, int64_t pos, int dim, int piece) {
    const bool ok = pos >= 0 && pos < p.max_positions;
    const int64_t lo = (ok ? pos : 0) * dim + piece * E, hi = lo + dim / 2;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      Chunk<float>::unpack(load16(p.cos_t + lo + e), cl + e);
      Chunk<float>::unpack(load16(p.sin_t + lo + e), sl + e);
      Chunk<float>::unpack(load16(p.cos_t + hi + e), ch + e);
      Chunk<float>::unpack(load16(p.sin_t + hi + e), sh + e);
    }
    if (!ok) {
#pragma unroll
      for (int e = 0; e < E; ++e) cl[e] = ch[e] = __int_as_float(0x7fc00000);
    }
  }
  __device__ void turn(float (&lo)[E], float (&hi)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float a = lo[e], b = hi[e];
      lo[e] = __fsub_rn(__fmul_rn(a, cl[e]), __fmul_rn(b, sl[e]));
      hi[e] = __fadd_rn(__fmul_rn(b, ch[e]), __fmul_rn(a, sh[e]));
    }
  }
};

template <typename TPos>
__device__ __forceinline__ int64_t position_of(const RopeWriteParams& p, int token) {
  return static_cast<int64_t>(static_cast<const TPos*>(p.positions)[token]);
}

// G heads of one token from `src` turned into `dst` (dst null: nothing is stored).
template <typename T, int G>
__device__ __forceinline__ void turn_heads(const RopeWriteParams& p, const char* src, char* dst,
                                           int64_t pos, int dim, int piece) {
  const int64_t row = static_cast<int64_t>(dim) * Elem<T>::kBytes, half = row / 2;
  Piece<T> lo[G], hi[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    lo[g].load(src + g * row);
    hi[g].load(src + g * row + half);
  }
  Angles a;
  a.load(p, pos, dim, piece);
  if (dst == nullptr) return;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float x[E], y[E];
    lo[g].unpack(x);
    hi[g].unpack(y);
    a.turn(x, y);
    lo[g].pack(x);
    hi[g].pack(y);
    lo[g].store(dst + g * row);
    hi[g].store(dst + g * row + half);
  }
}

// Pools of the inputs' type. Threads: (token, G heads of q, k or v, piece), pieces fastest.
template <typename T, typename TPos, int G>
__global__ __launch_bounds__(256) void rope_write_kernel(const RopeWriteParams p, int dim,
                                                         uint32_t pieces, uint32_t per_token,
                                                         uint32_t threads) {
  const uint32_t index = blockIdx.x * blockDim.x + threadIdx.x;
  if (index >= threads) return;
  const int token = static_cast<int>(index / per_token);
  const uint32_t rest = index - token * per_token;
  const int group = static_cast<int>(rest / pieces);
  const int piece = static_cast<int>(rest - group * pieces);
  const int head = group * G;
  constexpr int kBytes = Elem<T>::kBytes;
  const int64_t row = static_cast<int64_t>(dim) * kBytes;
  const int64_t in_row = static_cast<int64_t>(piece) * E * kBytes;
  if (head < p.hq) {
    const char* src = static_cast<const char*>(p.q) + (token * p.q_stride * kBytes + head * row + in_row);
    char* dst = static_cast<char*>(p.q_out) + ((static_cast<int64_t>(token) * p.hq + head) * row + in_row);
    turn_heads<T, G>(p, src, dst, position_of<TPos>(p, token), dim, piece);
    return;
  }
  const int32_t slot = p.slots[token];
  const bool held = slot >= 0 && slot < (p.num_blocks << p.block_shift);
  const bool is_v = head >= p.hq + p.hk;
  const int kvh = head - p.hq - (is_v ? p.hk : 0);
  const int64_t at = (static_cast<int64_t>(slot) * p.hk + kvh) * row + in_row;
  const char* src = static_cast<const char*>(is_v ? p.v : p.k) +
                    (token * (is_v ? p.v_stride : p.k_stride) * kBytes + kvh * row + in_row);
  if (is_v) {
    if (!held) return;
    Piece<T> lo[G], hi[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      lo[g].load(src + g * row);
      hi[g].load(src + g * row + row / 2);
    }
    char* dst = static_cast<char*>(p.v_pool) + at;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      lo[g].store(dst + g * row);
      hi[g].store(dst + g * row + row / 2);
    }
    return;
  }
  turn_heads<T, G>(p, src, held ? static_cast<char*>(p.k_pool) + at : nullptr,
                   position_of<TPos>(p, token), dim, piece);
}

// ---------------------------------------------------------------------- fp8

// Least power of two >= t (t >= 0 finite; 0 stays 0, a subnormal gives 2^-126).
__device__ __forceinline__ float pow2_at_least(float t) {
  const uint32_t b = __float_as_uint(t);
  if ((b & 0x7fffffu) == 0) return t;
  return __uint_as_float((b & 0x7f800000u) + 0x800000u);
}

// Eight values times `inv` (a power of two: exact) as e4m3 codes, saturating; NaN stays NaN.
__device__ __forceinline__ u32x2 encode8(const float (&x)[E], float inv) {
  auto at = [&](int e) __attribute__((always_inline)) {
    const float v = __fmul_rn(x[e], inv);
    return v > 448.0f ? 448.0f : (v < -448.0f ? -448.0f : v);
  };
  u32x2 out;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(at(4 * h), at(4 * h + 1), 0, false);
    out[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(at(4 * h + 2), at(4 * h + 3), lo, true));
  }
  return out;
}

// The largest magnitude among finite values (an infinity saturates and a NaN stays one: neither
// takes the page's other rows with it).
__device__ __forceinline__ float finite_max(float m, const float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float a = fabsf(x[e]);
    m = fmaxf(m, a < INFINITY ? a : 0.0f);
  }
  return m;
}

// Every `every`th workgroup while there are q_wgs: q, G heads a thread. The others: a window of tokens
// and a kv head, kRows tokens at a time, a row of threads each (K's pieces, then V's).
//   A window's workgroup writes the runs that start in it, all at once: the rows from its first start
// to the end of its last run, which may lie in the next window. Slots and positions are loaded once,
// a lane each, and handed round from there; runs are stretches of two bit masks; a run's maxima meet
// in LDS (the order of a maximum does not matter). So a run's rows, angles and old scale are
// requested one round trip after the launch, and 16 single tokens take as long as a page of 16.
// One run after another, each finding its slots, length, positions and angles in turn, and q's
// workgroups last: 9637 tokens in eight chunks 37.7 us, now 35.4 (4.2 TB/s); 128 tokens 10.3, now 6.5;
// 2048 single tokens 44.9, now 11.9; 64 level at 4.4.
template <typename T, typename TPos, int D, int G>
__global__ __launch_bounds__(256) void rope_write_fp8_kernel(const RopeWriteParams p, int every,
                                                             int q_wgs, uint32_t q_threads) {
  constexpr int kBytes = Elem<T>::kBytes;
  constexpr int kPieces = D / 2 / E;        // threads of a head vector
  constexpr int kRowThreads = 2 * kPieces;  // of a row: K's, then V's
  constexpr int kRows = 256 / kRowThreads;  // of a pass, and tokens of a window
  constexpr int64_t kRow = static_cast<int64_t>(D) * kBytes;
  static_assert(kRows <= kWave, "a window's tokens are held a lane each");
  const int bid = static_cast<int>(blockIdx.x);
  const int q_before = min(bid / every, q_wgs);
  if (q_before < q_wgs && bid % every == every - 1) {
    const uint32_t index = static_cast<uint32_t>(q_before) * 256 + threadIdx.x;
    if (index >= q_threads) return;
    const uint32_t per_token = static_cast<uint32_t>(p.hq / G) * kPieces;
    const int token = static_cast<int>(index / per_token);
    const uint32_t rest = index - token * per_token;
    const int head = static_cast<int>(rest / kPieces) * G;
    const int piece = static_cast<int>(rest % kPieces);
    const int64_t in_row = static_cast<int64_t>(piece) * E * kBytes;
    turn_heads<T, G>(p,
                     static_cast<const char*>(p.q) + (token * p.q_stride * kBytes + head * kRow + in_row),
                     static_cast<char*>(p.q_out) +
                         ((static_cast<int64_t>(token) * p.hq + head) * kRow + in_row),
                     position_of<TPos>(p, token), D, piece);
    return;
  }
  __shared__ uint32_t s_max[kRows][2];  // of the window's runs, the bits of a float >= 0
  __shared__ float s_old[kRows][2];     // their pages' scales before
  const int tid = threadIdx.x, lane = tid % kWave;
  const int head = (bid - q_before) % p.hk;
  const int first = (bid - q_before) / p.hk * kRows;
  const int my_row = tid / kRowThreads;
  const bool is_v = tid % kRowThreads >= kPieces;
  const int piece = tid % kPieces;

  // Lane i: token first + i. It starts a run when its slot is in the pool and does not continue the
  // slot of the token before on the same page.
  const int mine = min(first + lane, p.tokens - 1);
  const int my_slot = p.slots[mine];
  const TPos my_position = static_cast<const TPos*>(p.positions)[mine];
  const int slot_before = first > 0 ? p.slots[first - 1] : -1;
  const int up = __shfl_up(my_slot, 1, kWave);
  const int prev = lane > 0 ? up : slot_before;
  const bool live = first + lane < p.tokens && my_slot >= 0 && (my_slot >> p.block_shift) < p.num_blocks;
  const bool goes_on = live && prev >= 0 && prev + 1 == my_slot &&
                       (prev >> p.block_shift) == (my_slot >> p.block_shift);
  const uint64_t window = kRows == kWave ? ~uint64_t{0} : (uint64_t{1} << (kRows % kWave)) - 1;
  const uint64_t on = __builtin_amdgcn_ballot_w64(goes_on);
  const uint64_t starts = __builtin_amdgcn_ballot_w64(live && !goes_on) & window;
  if (starts == 0) return;  // the whole workgroup
  const int i0 = __builtin_ctzll(starts);
  // The last run's rows behind the window: lanes, then tokens past the lanes.
  int end = kRows;  // (a lane, or past them)
  while (end < kWave && (on >> (end % kWave) & 1)) ++end;
  if (end == kWave) {
    const int last = 63 - __builtin_clzll(starts);
    if (kRows < kWave || (on >> 63 & 1) || last == 63) {
      const int slot_last = __builtin_amdgcn_readlane(my_slot, last);
      const int room = (1 << p.block_shift) - (slot_last & ((1 << p.block_shift) - 1));
      for (bool more = true; more; ) {
        const int i = end + lane;
        const bool same = i - last < room && first + i < p.tokens && p.slots[first + i] == slot_last + i - last;
        const uint64_t not_same = __builtin_amdgcn_ballot_w64(!same);
        end += not_same != 0 ? __builtin_ctzll(not_same) : kWave;
        more = not_same == 0;
      }
    }
  }
  const int passes = (end - i0 + kRows - 1) / kRows;

  // This thread's row of a pass: its run, the run's first slot, and the row's token.
  int token = 0, run = 0, run_slot = 0, in_run = 0, run_rows = 0;
  int64_t position = 0;
  bool row = false;
  auto find = [&](int pass) __attribute__((always_inline)) {
    const int i = i0 + pass * kRows + my_row;
    const int at = min(i, kWave - 1);
    const uint64_t before = starts & (at == kWave - 1 ? ~uint64_t{0} : (uint64_t{2} << at) - 1);
    const int start = 63 - __builtin_clzll(before);  // (i0 is among them)
    run = __builtin_popcountll(before) - 1;
    row = i < end && (i >= kWave || ((starts | on) >> at & 1));
    token = first + i;
    in_run = i - start;
    const uint64_t stops = ~on & (start == kWave - 1 ? 0 : ~uint64_t{0} << (start + 1));
    const int stop = stops != 0 ? min(__builtin_ctzll(stops), end) : end;
    run_rows = stop - start;
    run_slot = __shfl(my_slot, start, kWave);
    const int low = __shfl(static_cast<int>(my_position), at, kWave);
    position = low;
    if constexpr (sizeof(TPos) == 8) {
      const int high = __shfl(static_cast<int>(static_cast<int64_t>(my_position) >> 32), at, kWave);
      position = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(high)) << 32 |
                                      static_cast<uint32_t>(low));
    }
    if (row && i >= kWave) position = position_of<TPos>(p, token);
  };
  float x[E], y[E];
  auto take = [&]() __attribute__((always_inline)) {  // the row, turned
    const char* src = static_cast<const char*>(is_v ? p.v : p.k) +
                      (token * (is_v ? p.v_stride : p.k_stride) * kBytes + head * kRow + piece * E * kBytes);
    Piece<T> lo, hi;
    lo.load(src);
    hi.load(src + kRow / 2);
    Angles a;
    if (!is_v) a.load(p, position, D, piece);
    lo.unpack(x);
    hi.unpack(y);
    if (!is_v) a.turn(x, y);
  };

  auto scale_at = [&]() __attribute__((always_inline)) -> float* {
    return (is_v ? p.v_scales : p.k_scales) +
           (static_cast<int64_t>(run_slot >> p.block_shift) * p.hk + head);
  };

  for (int i = tid; i < 2 * kRows; i += 256) s_max[i / 2][i % 2] = 0;
  __syncthreads();
  for (int pass = 0; pass < passes; ++pass) {
    find(pass);
    float most = 0.0f;
    if (row) {
      if (in_run == 0 && piece == 0) {
        s_old[run][is_v] = (run_slot & ((1 << p.block_shift) - 1)) != 0 ? *scale_at() : 0.0f;
      }
      take();
      most = finite_max(finite_max(0.0f, x), y);
    }
    most = group_max<kPieces>(most);
    if (row && piece == 0) atomicMax(&s_max[run][is_v], __float_as_uint(most));
  }
  __syncthreads();
  for (int pass = 0; pass < passes; ++pass) {
    if (passes > 1) {  // (else the row is held still)
      find(pass);
      if (row) take();
    }
    if (!row) continue;
    const float old = s_old[run][is_v];
    const float scale = fmaxf(old, pow2_at_least(__uint_as_float(s_max[run][is_v]) / 448.0f));
    const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;  // exact: a power of two
    const int64_t pool_row = static_cast<int64_t>(p.hk) * D;
    const int off0 = run_slot & ((1 << p.block_shift) - 1);
    uint8_t* pool = static_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) +
                    (static_cast<int64_t>(run_slot - off0) * p.hk + head) * D + piece * E;
    if (old > 0.0f && scale > old) {  // the page's earlier rows, shared out among the run's
      constexpr int kAhead = 4;
      for (int r0 = in_run; r0 < off0; r0 += kAhead * run_rows) {
        u32x2 w[kAhead][2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * run_rows < off0 ? r0 + u * run_rows : r0;
#pragma unroll
          for (int h = 0; h < 2; ++h) w[u][h] = *reinterpret_cast<const u32x2*>(pool + r * pool_row + h * (D / 2));
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * run_rows;
          if (r >= off0) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[E];
#pragma unroll
            for (int b = 0; b < E; ++b) {
              v[b] = __fmul_rn(fp8e4m3_to_f32((w[u][h][b / 4] >> (8 * (b % 4))) & 0xffu), old);
            }
            *reinterpret_cast<u32x2*>(pool + r * pool_row + h * (D / 2)) = encode8(v, inv);
          }
        }
      }
    }
    if (in_run == 0 && piece == 0) *scale_at() = scale;
    uint8_t* at = pool + (off0 + in_run) * pool_row;
    *reinterpret_cast<u32x2*>(at) = encode8(x, inv);
    *reinterpret_cast<u32x2*>(at + D / 2) = encode8(y, inv);
  }
}

// ----------------------------------------------------------------- dispatch

// Heads a thread takes: the largest of 4 and 2 that divides the head counts and leaves two waves
// per SIMD of 256 CUs, else 1.
int heads_per_thread(int64_t threads, int hq, int hk) {
  for (int g = 4; g > 1; g /= 2) {
    if (hq % g == 0 && hk % g == 0 && threads / g >= (int64_t{1} << 17)) return g;
  }
  return 1;
}

template <typename T, typename TPos>
hipError_t launch_same(const RopeWriteParams& p, int dim, hipStream_t stream) {
  const int64_t heads = p.hq + 2 * static_cast<int64_t>(p.hk);
  const int64_t pieces = dim / 2 / E;
  const int g = heads_per_thread(p.tokens * heads * pieces, p.hq, p.hk);
  const int64_t threads = p.tokens * (heads / g) * pieces;
  if (threads >= int64_t{1} << 31) return hipErrorInvalidValue;
  const unsigned bs = threads <= 65536 ? 64 : 256;
  const unsigned grid = static_cast<unsigned>((threads + bs - 1) / bs);
  const uint32_t per_token = static_cast<uint32_t>(heads / g * pieces);
#define MVLLM_ROPE_WRITE(G)                                                               \
  rope_write_kernel<T, TPos, G><<<grid, bs, 0, stream>>>(p, dim, static_cast<uint32_t>(pieces), \
                                                         per_token, static_cast<uint32_t>(threads))
  if (g == 4) MVLLM_ROPE_WRITE(4);
  else if (g == 2) MVLLM_ROPE_WRITE(2);
  else MVLLM_ROPE_WRITE(1);
#undef MVLLM_ROPE_WRITE
  return hipGetLastError();
}

template <typename T, typename TPos, int D>
hipError_t launch_fp8(const RopeWriteParams& p, hipStream_t stream) {
  constexpr int kPieces = D / 2 / E, kRows = 256 / (2 * kPieces);
  const int64_t kv_wgs = (p.tokens + kRows - 1) / kRows * static_cast<int64_t>(p.hk);
  const int64_t q_all = static_cast<int64_t>(p.tokens) * p.hq * kPieces;
  const int g = heads_per_thread(q_all, p.hq, p.hq);
  const int64_t q_threads = q_all / g;
  const int64_t q_wgs = (q_threads + 255) / 256, grid = kv_wgs + q_wgs;
  if (q_threads >= int64_t{1} << 31 || grid >= int64_t{1} << 31) return hipErrorInvalidValue;
  const int every = static_cast<int>(grid / q_wgs);  // (>= 1: every q_wgs-th position is in the grid)
#define MVLLM_ROPE_WRITE(G)                                                            \
  rope_write_fp8_kernel<T, TPos, D, G><<<static_cast<unsigned>(grid), 256, 0, stream>>>( \
      p, every, static_cast<int>(q_wgs), static_cast<uint32_t>(q_threads))
  if (g == 4) MVLLM_ROPE_WRITE(4);
  else if (g == 2) MVLLM_ROPE_WRITE(2);
  else MVLLM_ROPE_WRITE(1);
#undef MVLLM_ROPE_WRITE
  return hipGetLastError();
}

template <typename T, typename TPos>
hipError_t launch_t(const RopeWriteParams& p, int pool_dtype, int dim, hipStream_t stream) {
  if (pool_dtype != kFP8E4M3) return launch_same<T, TPos>(p, dim, stream);
  switch (dim) {
    case 32: return launch_fp8<T, TPos, 32>(p, stream);
    case 64: return launch_fp8<T, TPos, 64>(p, stream);
    case 128: return launch_fp8<T, TPos, 128>(p, stream);
    case 256: return launch_fp8<T, TPos, 256>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

template <typename T>
hipError_t launch_pos(const RopeWriteParams& p, int pool_dtype, int dim, int bytes, hipStream_t stream) {
  return bytes == 8 ? launch_t<T, int64_t>(p, pool_dtype, dim, stream)
                    : launch_t<T, int32_t>(p, pool_dtype, dim, stream);
}

}  // namespace

bool rope_write_supported(int dtype, int pool_dtype, int head_dim) {
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return false;
  if (pool_dtype == kFP8E4M3) return head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256;
  return pool_dtype == dtype && head_dim > 0 && head_dim <= 1024 && head_dim % (2 * E) == 0;
}

hipError_t launch_rope_write(const RopeWriteParams& p, int dtype, int pool_dtype, int head_dim,
                             int positions_bytes, hipStream_t stream) {
  switch (dtype) {
    case kF32: return launch_pos<float>(p, pool_dtype, head_dim, positions_bytes, stream);
    case kF16: return launch_pos<f16_t>(p, pool_dtype, head_dim, positions_bytes, stream);
    case kBF16: return launch_pos<bf16_t>(p, pool_dtype, head_dim, positions_bytes, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mvllm
