// Log-probabilities of given categories, entropy and likeliest categories of rows of scores: choice of the kernel, rows of any
// length and stride (score_stream_kernel).  Short rows and rows that lie side by side: category_scores_short.hip.
#include "category_stats.hip.hpp"

namespace pcm {

void check_rows(const RowsRef& x, const RowsShape& shape, const char* what) {
  if (shape.examples < 0 || shape.vars < 1 || shape.cats < 1)
    fail(PCM_ERR_SHAPE, "%s: %lld examples, %d variables, %d categories", what, (long long)shape.examples, shape.vars, shape.cats);
  if (shape.examples > INT64_C(0x7fffffff) / shape.vars) fail(PCM_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows", what);
  if (shape.cats > 1 << 30) fail(PCM_ERR_UNSUPPORTED, "%s: at most 2^30 categories", what);
  if (x.dtype != PCM_F32 && x.dtype != PCM_BF16 && x.dtype != PCM_F16) fail(PCM_ERR_ARG, "%s: type %d is none of PCM_F32, PCM_BF16, PCM_F16", what, x.dtype);
}

void check_given(const GivenRef& g) {
  if (g.slots < 0 || g.slots > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d given categories per row, got %d", kMaxSlots, g.slots);
  if (g.slots && !g.p) fail(PCM_ERR_ARG, "given categories: the pointer is null");
  if (g.slots && g.type != PCM_U8 && g.type != PCM_I32 && g.type != PCM_I64)
    fail(PCM_ERR_ARG, "given categories: type %d is none of PCM_U8, PCM_I32, PCM_I64", g.type);
}

namespace {
constexpr int kEntries = 16, kChunk = 64 * kEntries;   // of a lane, of a wave, at a time (32 entries of 2 bytes cost 20 spilled registers)
constexpr int kMaxWaves = 16, kMaxParts = 64;
constexpr int kRoom = 64;                   // common keys per wave of a workgroup
constexpr int kOneListChunks = 4;           // most chunks of a wave whose entries go into one list of the workgroup's
constexpr int kNoList = 0, kListPerWave = 1, kOneList = 2;

struct PartRef {                            // what parts of a row leave for the kernel that joins them
  float4* sums;                             // [rows][parts] m, s, t
  uint64_t* keys;                           // [rows][parts][top], falling
};

// How rows are dealt out: waves of a workgroup, and workgroups, per row
struct Split {
  int waves, parts, part_len;
};

// A wave's 64 likeliest entries so far, lane i holding the i-th as entry_key, and those that wait to be sorted in.  Entries at or
// below `bar`, the value of the top-th so far, are left out; what passes waits in LDS, and 64 at a time are sorted and merged.
// Groups of entries come by rising index, so that one that equals the bar of earlier groups loses to what is there.
struct TopList {
  uint64_t list = 0;
  float bar;
  int count = 0;
  // up to N waiting keys sorted, rising, into the last lanes
  template <int N>
  __device__ __forceinline__ uint64_t sorted(const uint64_t* wait) const {
    const int i = (int)(threadIdx.x & 63) - (64 - N);
    return sort_lanes<N, false>(i >= 0 && i < count ? wait[i] : (uint64_t)0);
  }
  __device__ __forceinline__ void flush(uint64_t* wait, int top) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
    const uint64_t k = count <= 16 ? sorted<16>(wait) : count <= 32 ? sorted<32>(wait) : sorted<64>(wait);
    list = sort_merge<64, true>(list > k ? list : k);
    const uint64_t rest = lane + 64 < count ? wait[lane + 64] : 0;
    __builtin_amdgcn_wave_barrier();
    if (lane + 64 < count) wait[lane] = rest;
    __builtin_amdgcn_wave_barrier();
    count = max(count - 64, 0);
    const uint32_t last = __builtin_amdgcn_readlane((uint32_t)(list >> 32), top - 1);
    if (last) bar = fmaxf(bar, order_float(last));
  }
  // the number just below one of float_order's (where both zeros are +0): a bar that the number itself passes
  static __device__ __forceinline__ float below(uint32_t order) { return order_float(order - (order == 0x80000000u ? 2 : 1)); }
};

// Writes the entries x of category c of the lanes in `some` behind the first `count` keys; returns how many there are then.
__device__ __forceinline__ int add_keys(uint64_t some, float x, uint32_t c, uint64_t* to, int count) {
  if (some >> (threadIdx.x & 63) & 1)
    to[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0))] = entry_key(x, c);
  return count + __popcll(some);
}

// the results of a row from its sums and sorted keys, by one wave
template <typename T>
__device__ __forceinline__ void write_row(const RowSums<T>& q, uint64_t key, int64_t r, int64_t e, int64_t v, const RowsRef& x, const RowsShape& shape,
                                          const GivenRef& given, int top, const ScoreOut& out) {
  const int lane = threadIdx.x & 63;
  const RowResult<T> res(q);
  const T* row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
  if (lane < given.slots)
    out.logp[r * given.slots + lane] = res.given(given_at(given, e, v, lane), shape.cats, [&](int64_t g) { return seen(row[g * x.stride_cat]); });
  if (lane == 0) {
    if (out.log_sum) out.log_sum[r] = res.log_sum();
    if (out.entropy) out.entropy[r] = res.entropy(q);
  }
  if (lane < top) {
    out.top[r * top + lane] = res.nan || !key ? -1 : key_index(key);
    out.top_logp[r * top + lane] = res.nan ? NAN : !key ? -INFINITY : res.logp(key_value(key));
  }
}

// One pass over a row, or a part of it, by the waves of a workgroup.  A wave takes kEntries a lane at a time (16 bytes a request, one
// entry at a time where categories are not neighbours), requests the ones after the next as soon as these are in float, and keeps one maximum
// for its lanes: a group whose largest entry lies above neither the maximum nor the list's bar goes straight into the sums.
// 4096 rows of 131072 bf16 with entropy: 184 us without a list, 5.8 TB/s, 201 with the 8 likeliest (reads alone reach 7; about 10 instruction
// slots an entry, the exponential four of them, are 130 us); 2048 rows of 32003 f32 with 16 given and 16 likeliest: 57 us, 4.6 TB/s;
// with a checkpoint, 4096 of 50304 bf16: 148 us, 4.3 TB/s read and written.
template <typename T, bool kUnit, bool kEnt, int kLists, bool kCkpt>
__global__ __launch_bounds__(64 * kMaxWaves) void score_stream_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, CkptRef ckpt,
                                                                      int parts, int part_len, PartRef part) {
  constexpr bool kTop = kLists != kNoList, kCommon = kLists == kOneList;
  constexpr int kVec = kUnit ? 16 / (int)sizeof(T) : 1, kLoads = kEntries / kVec;
  extern __shared__ uint64_t stream_lds[];   // per wave 128 keys that wait, and its sums; the common keys
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  uint64_t* const wait = stream_lds + 128 * wave;
  float4* const sums_lds = reinterpret_cast<float4*>(stream_lds + 128 * waves);
  uint64_t* const ours = reinterpret_cast<uint64_t*>(sums_lds + waves);   // the waves' common keys
  const int room = kRoom * waves;
  __shared__ uint32_t seed[kCommon ? 256 : 1];
  __shared__ int ours_count, ours_full, crowds;
  __shared__ float ours_bar;
  const int64_t jobs = shape.rows() * parts;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;

  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const uint32_t r = parts == 1 ? (uint32_t)job : (uint32_t)job / (uint32_t)parts;   // (more than one part: fewer than 2^31 jobs)
    const int q = parts == 1 ? 0 : (int)((uint32_t)job - r * (uint32_t)parts);
    const int64_t e = shape.vars == 1 ? r : r / (uint32_t)shape.vars, v = shape.vars == 1 ? 0 : r % (uint32_t)shape.vars;
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    const int first = q * part_len, end = parts == 1 ? shape.cats : min(first + part_len, shape.cats);

    RowSums<T> sum;
    TopList list;
    list.bar = masked_from<T>();
    bool fresh = !kCommon;

    struct Chunk { typename std::conditional<kUnit, raw4, T>::type g[kLoads]; };
    auto load = [&](Chunk& k, int at) {                       // a whole chunk
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        if constexpr (kUnit) k.g[u] = load16(row + at + (u * 64 + lane) * kVec);
        else k.g[u] = row[(int64_t)(at + u * 64 + lane) * x.stride_cat];
      }
    };
    auto load_end = [&](Chunk& k, int at) {                   // the first or the last one: -inf before the start and behind the end
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int c = at + (u * 64 + lane) * kVec;
        if constexpr (kUnit) {
          if (c >= first && c + kVec <= end) k.g[u] = load16(row + c);
          else {
            T w[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) w[i] = c + i >= first && c + i < end ? row[c + i] : (T)-INFINITY;
            k.g[u] = __builtin_bit_cast(raw4, w);
          }
        } else k.g[u] = c < end ? row[(int64_t)c * x.stride_cat] : (T)-INFINITY;
      }
    };
    auto entries = [&](const Chunk& k, int u, float (&y)[kVec]) {
      if constexpr (kUnit) unpack(k.g[u], y, T());
      else y[0] = seen(k.g[u]);
    };
    // Entries of two bytes: requests at multiples of 16 bytes, so that none straddles two lines (4096 rows of 50303: 97 us without, 75 of 50304).
    // A checkpoint's blocks begin with the row.
    const int start = kUnit && !kCkpt && sizeof(T) == 2 ? first - (int)((uintptr_t)(row + first) % 16 / sizeof(T)) : first;
    const int chunks = (end - start + kChunk - 1) / kChunk;
    auto request = [&](Chunk& k, int j) {
      const int at = start + j * kChunk;
      if (at >= first && at + kChunk <= end) load(k, at);
      else if (j < chunks) load_end(k, at);
    };
    auto work = [&](Chunk& k, int j) {
      const int at = start + j * kChunk;
      float y[kLoads][kVec], largest[kLoads], lane_largest = -INFINITY;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        entries(k, u, y[u]);
        largest[u] = y[u][0];
#pragma unroll
        for (int i = 1; i < kVec; ++i) largest[u] = __builtin_elementwise_maximum(largest[u], y[u][i]);
        lane_largest = __builtin_elementwise_maximum(lane_largest, largest[u]);
      }
      request(k, j + 2 * waves);
      if (kTop && fresh) {
        // the top-th largest of the lanes' largest entries is no larger than the top-th largest entry: a bar to start from
        const uint32_t last = __builtin_amdgcn_readlane(sort_lanes<64, true>(float_order(lane_largest)), top - 1);
        list.bar = fmaxf(list.bar, TopList::below(last));
        fresh = false;
      }
      if (__any(lane_largest > (kTop ? fminf(list.bar, sum.m) : sum.m))) {   // (another wave's entries may have set the bar)
        if (!kTop || __any(lane_largest > sum.m)) {
          const float m1 = over_lanes<64>(lane_largest, Larger());
          if (m1 > sum.m) sum.raise(m1);
        }
        if constexpr (kTop) {
          const float above = list.bar;           // (the bar of earlier chunks, also where it rises in between)
          const int early = max(top, 16);         // that many waiting entries are sorted in at once, so that the bar rises
          uint32_t crowded = 0;                   // groups with more entries above the bar than there is room for
#pragma unroll
          for (int u = 0; u < kLoads; ++u)
            if (__any(largest[u] > above)) {
              uint64_t some[kVec];
              int all = 0;
#pragma unroll
              for (int i = 0; i < kVec; ++i) all += __popcll(some[i] = __ballot(y[u][i] > above));
              // with several waves into the common keys, where there is room
              uint64_t* to = wait;
              int count = list.count, most = 128;
              if (kCommon) {
                if (lane == 0) {
                  count = atomicAdd(&ours_count, all);
                  if (count + all > room) atomicMin(&ours_full, count);
                }
                count = __builtin_amdgcn_readfirstlane(count);
                to = ours;
                most = room;
              }
              if (count + all > most) crowded |= 1u << u;
              else {
                if (!kCommon) list.count += all;
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                  if (some[i]) count = add_keys(some[i], y[u][i], (uint32_t)(at + (u * 64 + lane) * kVec + i), to, count);
              }
            }
          // what is full is sorted in, then the crowded groups' entries are added, one of every lane at a time
          uint32_t hit = 0;
          float z[kVec];
          int zc = 0;
          for (;;) {
            const uint64_t some = __ballot(hit != 0);
            if (list.count >= (some || crowded ? 64 : early)) list.flush(wait, top);
            else if (some) {
              const int i = hit ? __builtin_ctz(hit) : 0;
              float v = z[0];
#pragma unroll
              for (int j = 1; j < kVec; ++j) v = i == j ? z[j] : v;
              list.count = add_keys(some, v, (uint32_t)(zc + i), wait, list.count);
              hit &= hit - 1;
            } else if (crowded) {
              const int u = __builtin_ctz(crowded);
              crowded &= crowded - 1;
#pragma unroll
              for (int w = 0; w < kLoads; ++w)
                if (u == w)
#pragma unroll
                  for (int i = 0; i < kVec; ++i) z[i] = y[w][i];
              zc = at + (u * 64 + lane) * kVec;
              if (kCommon) crowds = 1;
#pragma unroll
              for (int i = 0; i < kVec; ++i) hit |= z[i] > above ? 1u << i : 0u;
            } else break;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        if (at + u * 64 * kVec >= end) break;
        float gs = 0.f, gt = 0.f;
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum.template add<kEnt>(y[u][i], gs, gt);
        sum.s += gs;
        sum.t += gt;
        if constexpr (kCkpt) {
          const int c = at + (u * 64 + lane) * kVec;
          store_codes(ckpt, encode_block<T>(y[u]), r, c, shape.cats, pitch, blocks);
        }
      }
    };

    Chunk even, odd;
    request(even, wave);
    request(odd, wave + waves);
    if constexpr (kCommon) {
      // One bar for all waves: the top-th largest, to 16 bits, of the largest entries of up to 256 sets of lanes.  The row's likeliest
      // entries lie above it, and not many more: the waves collect them together, and one of them sorts them in the end.
      const int sets = waves <= 4 ? 64 : 256 / waves, each = 64 / sets, words = sets * waves / 64;
      float largest = -INFINITY;
      if (wave < chunks) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          float y[kVec];
          entries(even, u, y);
#pragma unroll
          for (int i = 0; i < kVec; ++i) largest = __builtin_elementwise_maximum(largest, y[i]);
        }
      }
      if (each > 1) largest = fmaxf(largest, dpp<0xB1>(largest));
      if (each > 2) largest = fmaxf(largest, dpp<0x4E>(largest));
      if (lane % each == 0) seed[wave * sets + lane / each] = float_order(largest);
      __syncthreads();
      if (wave == 0) {
        uint32_t v[4], bar = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < words ? seed[i * 64 + lane] : 0;
        for (int b = 31; b >= 16; --b) {
          const uint32_t higher = bar | 1u << b;
          int n = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) n += __popcll(__ballot(v[i] >= higher));
          if (n >= top) bar = higher;
        }
        if (lane == 0) {
          ours_bar = TopList::below(bar);
          ours_count = 0;
          ours_full = room;
          crowds = 0;
        }
      }
      __syncthreads();
      list.bar = fmaxf(list.bar, ours_bar);
    }
    for (int j = wave; j < chunks; j += 2 * waves) {
      work(even, j);
      if (j + waves < chunks) work(odd, j + waves);
    }
    if (kTop && list.count) list.flush(wait, top);   // (fewer than 64)
    sum.s = over_lanes<64>(sum.s, Sum());
    if (kEnt) sum.t = over_lanes<64>(sum.t, Sum());

    if (waves > 1) {
      if (lane == 0) sums_lds[wave] = make_float4(sum.m, sum.s, sum.t, 0.f);
      __syncthreads();
      if (kTop && (!kCommon || crowds)) {          // (one list: only of rows whose entries rise and rise)
        wait[lane] = list.list;
        __syncthreads();
        for (int h = waves >> 1; h > 0; h >>= 1) {   // two lists into one, the second one turned round
          if (wave < h) {
            const uint64_t k = stream_lds[128 * (wave + h) + 63 - lane];
            list.list = sort_merge<64, true>(list.list > k ? list.list : k);
            wait[lane] = list.list;
          }
          __syncthreads();
        }
      }
      if (kCommon && wave == 0) {
        const int all = min(ours_count, ours_full);
        for (int n = 0; n < all; n += 64) {
          list.count = min(all - n, 64);
          list.flush(ours + n, top);
        }
      }
      if (wave == 0) sum.join_lanes(lane < waves ? sums_lds[lane] : make_float4(masked_from<T>(), 0.f, 0.f, 0.f));
    }
    if (wave == 0) {
      if (parts == 1) write_row(sum, list.list, r, e, v, x, shape, given, top, out);
      else {
        if (lane == 0) part.sums[job] = make_float4(sum.m, sum.s, sum.t, 0.f);
        if (kTop && lane < top) part.keys[job * top + lane] = list.list;
      }
    }
    if (waves > 1) __syncthreads();   // the next row's keys go where these are read
  }
}

// The parts of a row put together, by a workgroup of four waves: 4.3 us, a launch and four merges of lists one after the other
template <typename T>
__global__ __launch_bounds__(256) void score_join_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, int parts, PartRef part) {
  __shared__ uint64_t keys[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t r = blockIdx.x;
  const int64_t e = r / (uint32_t)shape.vars, v = r % (uint32_t)shape.vars;
  RowSums<T> sum;
  const float4 own = lane < parts ? part.sums[(int64_t)r * parts + lane] : make_float4(masked_from<T>(), 0.f, 0.f, 0.f);
  uint64_t list = 0;
  if (top) {
    const int from = 63 - lane;
    uint64_t k[kMaxParts / 4];
#pragma unroll
    for (int i = 0; i < kMaxParts / 4; ++i) {   // all requests first
      const int p = wave + 4 * i;
      k[i] = p < parts && from < top ? part.keys[((int64_t)r * parts + p) * top + from] : 0;
    }
#pragma unroll
    for (int i = 0; i < kMaxParts / 4; ++i)
      if (wave + 4 * i < parts) list = sort_merge<64, true>(list > k[i] ? list : k[i]);
    keys[wave][lane] = list;
    __syncthreads();
    if (wave == 0)
      for (int w = 1; w < 4; ++w) {
        const uint64_t k = keys[w][from];
        list = sort_merge<64, true>(list > k ? list : k);
      }
  }
  if (wave == 0) {
    sum.join_lanes(own);
    write_row(sum, list, r, e, v, x, shape, given, top, out);
  }
}

// Rows that are fewer than keep the memory busy get several waves, up to one for every chunk: of one workgroup, which joins them in
// LDS, or of several, with a second launch to put the parts together.  Waves cost little where there are only sums (4096 rows of
// 131072 bf16 scores: 203 us with one wave a row, 184 with four, 230 with sixteen); a list of the likeliest costs each of them its start
// (8 likeliest: 206, 245 with two waves a row; 1000 rows of 50021 with 20: 71 with four, 90 with eight).
Split split_of(const RowsShape& shape, bool top) {
  const int64_t rows = shape.rows(), chunks = (shape.cats + kChunk - 1) / kChunk;
  const int64_t wanted = std::min(((top ? 2560 : 16384) + rows - 1) / rows, chunks);
  const int most = top ? kMaxWaves / 2 : kMaxWaves;
  Split s{1, 1, shape.cats};
  if (wanted <= 2 * most) {
    while (s.waves < std::min<int64_t>(wanted, most)) s.waves *= 2;
    return s;
  }
  s.waves = wanted > 8 * kMaxParts ? kMaxWaves : 8;
  const int64_t parts = std::min<int64_t>(kMaxParts, (wanted + s.waves - 1) / s.waves);
  s.part_len = (int)((chunks + parts - 1) / parts * kChunk);
  s.parts = (int)((shape.cats + s.part_len - 1) / s.part_len);
  return s;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

template <typename T>
void launch_stream(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt, void* work,
                   hipStream_t stream) {
  if (category_scores_short<T>(x, shape, given, top, out, ckpt, stream)) return;
  const Split s = split_of(shape, top > 0);
  PartRef part{};
  if (s.parts > 1) {
    part.sums = static_cast<float4*>(work);
    part.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(work) + up16((size_t)shape.rows() * s.parts * sizeof(float4)));
  }
  const dim3 grid((unsigned)std::min<int64_t>(shape.rows() * s.parts, 1 << 20)), block(64 * s.waves);
  const bool ent = out.entropy != nullptr;
  // A list of the likeliest per wave pays over many chunks, as its bar rises; one of all waves costs each of them little
  const int lists = !top ? kNoList : s.waves > 1 && s.part_len <= (int64_t)kOneListChunks * s.waves * kChunk ? kOneList : kListPerWave;
  const int lds = s.waves * (128 * 8 + 16 + (lists == kOneList ? kRoom * 8 : 0));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, lds, stream, x, shape, given, top, out, ckpt, s.parts, s.part_len, part); };
  auto choose = [&](auto unit, auto keep) {
    constexpr bool kUnit = decltype(unit)::value, kCkpt = decltype(keep)::value;
    if (lists == kNoList) ent ? launch(score_stream_kernel<T, kUnit, true, kNoList, kCkpt>) : launch(score_stream_kernel<T, kUnit, false, kNoList, kCkpt>);
    else if (lists == kListPerWave) ent ? launch(score_stream_kernel<T, kUnit, true, kListPerWave, kCkpt>) : launch(score_stream_kernel<T, kUnit, false, kListPerWave, kCkpt>);
    else ent ? launch(score_stream_kernel<T, kUnit, true, kOneList, kCkpt>) : launch(score_stream_kernel<T, kUnit, false, kOneList, kCkpt>);
  };
  if (x.stride_cat != 1) choose(std::false_type(), std::false_type());
  else if (ckpt.codes) choose(std::true_type(), std::true_type());
  else choose(std::true_type(), std::false_type());
  if (s.parts > 1)
    hipLaunchKernelGGL((score_join_kernel<T>), dim3((unsigned)shape.rows()), dim3(256), 0, stream, x, shape, given, top, out, s.parts, part);
}
}  // namespace

int64_t category_scores_workspace(const RowsShape& shape, int top) {
  if (shape.examples < 1 || shape.vars < 1 || shape.cats < 1 || shape.cats > 1 << 30 || top < 0 || top > kMaxSlots ||
      shape.examples > INT64_C(0x7fffffff) / shape.vars)
    return 0;
  const Split s = split_of(shape, top > 0);
  const size_t jobs = (size_t)shape.rows() * s.parts;
  return s.parts == 1 ? 0 : (int64_t)(up16(jobs * sizeof(float4)) + jobs * top * sizeof(uint64_t));
}

void category_scores(const RowsRef& x_in, const RowsShape& shape_in, const GivenRef& given, int top, float* d_logp, float* d_log_sum,
                     float* d_entropy, float* d_top_logp, int32_t* d_top, const CkptRef& ckpt, void* d_work, int64_t work_bytes, hipStream_t stream) {
  check_rows(x_in, shape_in, "scores");
  check_given(given);
  if (top < 0 || top > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d likeliest categories, got %d", kMaxSlots, top);
  if (!ckpt.codes != !ckpt.scales) fail(PCM_ERR_ARG, "a checkpoint needs both its codes and its scales");
  if (!shape_in.examples) return;
  if (!x_in.p || (given.slots && !d_logp) || (top && (!d_top || !d_top_logp))) fail(PCM_ERR_ARG, "scores: a pointer is null");
  const int64_t need = category_scores_workspace(shape_in, top);
  if (need && (!d_work || work_bytes < need)) fail(PCM_ERR_ARG, "scores: %lld bytes of workspace, got %lld", (long long)need, (long long)work_bytes);
  if (((uintptr_t)d_work | (uintptr_t)ckpt.codes) & 15) fail(PCM_ERR_ARG, "scores: workspace and codes must be 16-byte aligned");
  RowsRef x = x_in;
  const RowsShape shape = shape_in;
  if (shape.cats == 1) x.stride_cat = 1;
  const ScoreOut out{d_logp, d_log_sum, d_entropy, d_top_logp, d_top};
  const CkptRef fused = x.stride_cat == 1 ? ckpt : CkptRef{};
  if (x.dtype == PCM_F32) launch_stream<float>(x, shape, given, top, out, fused, d_work, stream);
  else if (x.dtype == PCM_BF16) launch_stream<bf16>(x, shape, given, top, out, fused, d_work, stream);
  else launch_stream<f16>(x, shape, given, top, out, fused, d_work, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of category_scores failed: %s", hipGetErrorString(e));
  if (ckpt.codes && !fused.codes) checkpoint_rows(x, shape, ckpt, stream);
}

}  // namespace pcm
