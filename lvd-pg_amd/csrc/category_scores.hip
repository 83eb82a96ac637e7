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
constexpr int kGroups = 4;                  // 16-byte groups that a lane requests at a time
constexpr int kMaxWaves = 16, kMaxParts = 64;

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
  // those of a lane's entries y, of categories c.., that lie above the bar
  template <int N>
  __device__ __forceinline__ void take(const float (&y)[N], uint32_t c, uint64_t* wait, int top) {
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) hit |= y[i] > bar ? 1u << i : 0u;
    for (;;) {                                    // one entry of every lane that has some left
      const uint64_t some = __ballot(hit != 0);
      if (!some) break;
      if (hit) {
        const int i = __builtin_ctz(hit);
        float v = y[0];
#pragma unroll
        for (int j = 1; j < N; ++j) v = i == j ? y[j] : v;
        wait[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0))] = entry_key(v, c + i);
        hit &= hit - 1;
      }
      count += __popcll(some);
      // (64 fill what is sorted at a time; fewer are sorted in at the end of a group, so that the bar rises early)
      if (count >= 64 || (count >= max(top, 16) && !__any(hit != 0))) flush(wait, top);
    }
  }
};

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

// One pass over a row, or a part of it, by the waves of a workgroup.  A wave takes kGroups x 16 bytes a lane at a time (one
// entry at a time where categories are not neighbours), requests the next ones before it works on these, and keeps one maximum
// for its lanes: a group whose largest entry lies above neither the maximum nor the list's bar goes straight into the sums.
template <typename T, bool kUnit, bool kEnt, bool kTop, bool kCkpt>
__global__ __launch_bounds__(64 * kMaxWaves) void score_stream_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, CkptRef ckpt,
                                                                      int parts, int part_len, PartRef part) {
  constexpr int kVec = kUnit ? 16 / (int)sizeof(T) : 1, kLoads = kUnit ? kGroups : 16, kChunk = 64 * kVec * kLoads;
  extern __shared__ uint64_t stream_lds[];   // per wave 128 keys that wait, and its sums
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  uint64_t* const wait = stream_lds + 128 * wave;
  float4* const sums_lds = reinterpret_cast<float4*>(stream_lds + 128 * waves);
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
    bool fresh = true;

    struct Chunk { typename std::conditional<kUnit, raw4, T>::type g[kLoads]; };
    auto load = [&](Chunk& k, int at) {                       // a whole chunk
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        if constexpr (kUnit) k.g[u] = load16(row + at + (u * 64 + lane) * kVec);
        else k.g[u] = row[(int64_t)(at + u * 64 + lane) * x.stride_cat];
      }
    };
    auto load_end = [&](Chunk& k, int at) {                   // the last one: -inf behind the end
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int c = at + (u * 64 + lane) * kVec;
        if constexpr (kUnit) {
          if (c + kVec <= end) k.g[u] = load16(row + c);
          else {
            T w[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) w[i] = c + i < end ? row[c + i] : (T)-INFINITY;
            k.g[u] = __builtin_bit_cast(raw4, w);
          }
        } else k.g[u] = c < end ? row[(int64_t)c * x.stride_cat] : (T)-INFINITY;
      }
    };
    auto entries = [&](const Chunk& k, int u, float (&y)[kVec]) {
      if constexpr (kUnit) unpack(k.g[u], y, T());
      else y[0] = seen(k.g[u]);
    };
    auto work = [&](const Chunk& k, int at) {
      float y[kLoads][kVec], largest[kLoads], lane_largest = -INFINITY;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        entries(k, u, y[u]);
        largest[u] = y[u][0];
#pragma unroll
        for (int i = 1; i < kVec; ++i) largest[u] = __builtin_elementwise_maximum(largest[u], y[u][i]);
        lane_largest = __builtin_elementwise_maximum(lane_largest, largest[u]);
      }
      if (kTop && fresh) {
        // the top-th largest of the lanes' largest entries is no larger than the top-th largest entry: a bar to start from
        const uint32_t last = __builtin_amdgcn_readlane(sort_lanes<64, true>(float_order(lane_largest)), top - 1);
        list.bar = fmaxf(list.bar, order_float(last - (last == 0x80000000u ? 2 : 1)));   // (just below, both zeros being one: the entry itself has to pass)
        fresh = false;
      }
      if (__any(lane_largest > (kTop ? list.bar : sum.m))) {
        if (!kTop || __any(lane_largest > sum.m)) {
          const float m1 = over_lanes<64>(lane_largest, Larger());
          if (m1 > sum.m) sum.raise(m1);
        }
        if constexpr (kTop) {
          uint32_t groups = 0;                    // that have an entry above the bar
#pragma unroll
          for (int u = 0; u < kLoads; ++u) groups |= __any(largest[u] > list.bar) ? 1u << u : 0u;
          while (groups) {
            const int u = __builtin_ctz(groups);
            groups &= groups - 1;
            auto g = k.g[0];
#pragma unroll
            for (int w = 1; w < kLoads; ++w)
              if (u == w) g = k.g[w];
            float z[kVec];
            if constexpr (kUnit) unpack(g, z, T());
            else z[0] = seen(g);
            list.take(z, (uint32_t)(at + (u * 64 + lane) * kVec), wait, top);
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

    const int whole = (end - first) / kChunk, chunks = (end - first + kChunk - 1) / kChunk;
    Chunk now, next;
    auto request = [&](Chunk& k, int j) {
      if (j < whole) load(k, first + j * kChunk);
      else if (j < chunks) load_end(k, first + j * kChunk);
    };
    request(now, wave);
    for (int j = wave; j < chunks; j += waves) {
      request(next, j + waves);
      work(now, first + j * kChunk);
      now = next;
    }
    if (kTop && list.count) list.flush(wait, top);
    sum.s = over_lanes<64>(sum.s, Sum());
    if (kEnt) sum.t = over_lanes<64>(sum.t, Sum());

    if (waves > 1) {
      if (lane == 0) sums_lds[wave] = make_float4(sum.m, sum.s, sum.t, 0.f);
      if (kTop) wait[lane] = list.list;
      __syncthreads();
      if (kTop)
        for (int h = waves >> 1; h > 0; h >>= 1) {   // two lists into one, the second one turned round
          if (wave < h) {
            const uint64_t k = stream_lds[128 * (wave + h) + 63 - lane];
            list.list = sort_merge<64, true>(list.list > k ? list.list : k);
            wait[lane] = list.list;
          }
          __syncthreads();
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

// The parts of a row put together, by a workgroup of four waves
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

// Waves that keep the memory busy: 4096.  Rows that are fewer get several, up to one for every chunk of 64 x kGroups x 16 bytes: of one
// workgroup, which joins them in LDS, or, beyond 16, of several, with a second launch to put the parts together.
Split split_of(const RowsShape& shape, int entry_bytes) {
  const int64_t rows = shape.rows(), chunk = 64 * kGroups * 16 / entry_bytes, chunks = (shape.cats + chunk - 1) / chunk;
  const int64_t wanted = std::min((4096 + rows - 1) / rows, chunks);
  Split s{1, 1, shape.cats};
  if (wanted <= kMaxWaves) {
    while (s.waves < wanted) s.waves *= 2;
    return s;
  }
  s.waves = wanted > 8 * kMaxParts ? kMaxWaves : 8;
  const int64_t parts = std::min<int64_t>(kMaxParts, (wanted + s.waves - 1) / s.waves);
  s.part_len = (int)((chunks + parts - 1) / parts * chunk);
  s.parts = (int)((shape.cats + s.part_len - 1) / s.part_len);
  return s;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

template <typename T>
void launch_stream(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt, void* work,
                   hipStream_t stream) {
  if (category_scores_short<T>(x, shape, given, top, out, ckpt, stream)) return;
  const Split s = split_of(shape, sizeof(T));
  PartRef part{};
  if (s.parts > 1) {
    part.sums = static_cast<float4*>(work);
    part.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(work) + up16((size_t)shape.rows() * s.parts * sizeof(float4)));
  }
  const dim3 grid((unsigned)std::min<int64_t>(shape.rows() * s.parts, 1 << 20)), block(64 * s.waves);
  const int lds = s.waves * (128 * 8 + 16);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, lds, stream, x, shape, given, top, out, ckpt, s.parts, s.part_len, part); };
  const bool ent = out.entropy != nullptr;
  if (x.stride_cat != 1) {
    if (top) ent ? launch(score_stream_kernel<T, false, true, true, false>) : launch(score_stream_kernel<T, false, false, true, false>);
    else ent ? launch(score_stream_kernel<T, false, true, false, false>) : launch(score_stream_kernel<T, false, false, false, false>);
  } else if (ckpt.codes) {
    if (top) ent ? launch(score_stream_kernel<T, true, true, true, true>) : launch(score_stream_kernel<T, true, false, true, true>);
    else ent ? launch(score_stream_kernel<T, true, true, false, true>) : launch(score_stream_kernel<T, true, false, false, true>);
  } else {
    if (top) ent ? launch(score_stream_kernel<T, true, true, true, false>) : launch(score_stream_kernel<T, true, false, true, false>);
    else ent ? launch(score_stream_kernel<T, true, true, false, false>) : launch(score_stream_kernel<T, true, false, false, false>);
  }
  if (s.parts > 1)
    hipLaunchKernelGGL((score_join_kernel<T>), dim3((unsigned)shape.rows()), dim3(256), 0, stream, x, shape, given, top, out, s.parts, part);
}
}  // namespace

// (whatever the type and the strides: what the entries of four bytes need, or those of two)
int64_t category_scores_workspace(const RowsShape& shape, int top) {
  if (shape.examples < 1 || shape.vars < 1 || shape.cats < 1 || top < 0 || top > kMaxSlots || shape.examples > INT64_C(0x7fffffff) / shape.vars) return 0;
  int64_t most = 0;
  for (int bytes = 2; bytes <= 4; bytes += 2) {
    const Split s = split_of(shape, bytes);
    const size_t jobs = (size_t)shape.rows() * s.parts;
    if (s.parts > 1) most = std::max(most, (int64_t)(up16(jobs * sizeof(float4)) + jobs * top * sizeof(uint64_t)));
  }
  return most;
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
