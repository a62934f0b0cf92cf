// Layer norm over rows: y = (x - mean) rstd w + b, and its backward pass.
//
// Rows come in by bulk copies, several ahead of the one that is worked on, into a ring in shared memory; T threads (a warp,
// or a block) have a row, K groups of eight values each.  Forward: mean first, then the squares of what is left of the
// values (no difference of large sums), which are in registers meanwhile.  The backward pass takes x and dy,
//   h = (x - mean) rstd,  dx = rstd (w dy - mean(w dy) - h mean(w dy h)),  dw = sum dy h,  db = sum dy,
// twice from the ring, and has the column sums of a thread's own columns in its registers over all rows that its block
// works on.  Rows whose length eight does not divide begin at one of eight places within an aligned group; a block takes rows
// that begin at the same place, so that its threads keep their columns, whose w and b wait in shared memory.  The sums of the
// blocks are added by a second kernel in a fixed order.  Both passes should be bound by memory (18 and 28 us for 6001 x 5003
// values of bf16), which takes some 60 KB an SM on their way: with one row ahead in registers they took 104 and 109 us.  They take
// 32 and 53 now, at 40 % of the issue slots of 16 warps an SM, which wait for shared memory and for their team.
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

struct NormParams {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* out;       // y, or dx
  float* stats;    // [rows][2]: mean, rstd
  float* partial;  // backward: [block][2][width]
  int64_t rows, width;
  float eps;
  int param_type;
  int period;  // rows r, r + period, ... begin at the same place of an aligned group
  int stages, stage_bytes, x_bytes;  // of a ring: rows, bytes of a row's place, of its part that is x
};

__device__ unsigned int g_norm_status;

// A block stays on its SM for all rows; its teams of T threads share the parameters.  Forward with up to three groups a thread
// needs few registers, and its threads fill the SM; with more, or the column sums of the backward pass, half as many do.
template <int T, int K, bool kBackward>
struct Block {
  static constexpr int kThreads = kBackward || K > 3 ? 512 : 1024;
  static constexpr int kTeams = kThreads / T;
};
constexpr int kNormSmem = 220 * 1024;
constexpr int kMostStages = 8;

// eight values as four pairs
template <typename T>
__device__ __forceinline__ void load_pairs(const T* p, Pair (&v)[4]) {
  float f[8];
  load8(p, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pair(f[2 * j], f[2 * j + 1]);
}
// w and b wait in shared memory by place, in two halves: the first four of every group of eight, and the others.  (With eight
// neighbours a thread, every second thread of a warp met another one's banks: 6001 x 5003 bf16 forward 37 us, 32 this way.)
template <int kPlaces>
__device__ __forceinline__ int param_place(int i) {
  return (i >> 2 & 1) * (kPlaces / 2) + (i >> 3) * 4 + (i & 3);
}
template <int kPlaces>
__device__ __forceinline__ void load_params(const float* params, int group, Pair (&v)[4]) {
  const float4 a = reinterpret_cast<const float4*>(params)[group], b = reinterpret_cast<const float4*>(params + kPlaces / 2)[group];
  v[0] = pair(a.x, a.y), v[1] = pair(a.z, a.w), v[2] = pair(b.x, b.y), v[3] = pair(b.z, b.w);
}

// Of a thread's K groups only the first one can begin before the row, and only the last one end behind it, or the one before that
// where the row has no last one (it has a group less where it begins with a whole one).
template <int K>
__device__ __forceinline__ bool cut(int k, int first, int width) {
  return (k == 0 && first < 0) || (k >= K - 2 && first + 8 > width);
}
// zeros in the places of values that are not in [0, width)
template <int K>
__device__ __forceinline__ void keep_pairs(int k, Pair (&v)[4], int first, int width) {
  if (!cut<K>(k, first, width)) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    parts(v[j], a, b);
    const int c = first + 2 * j;
    v[j] = pair(c >= 0 && c < width ? a : 0.0f, c + 1 >= 0 && c + 1 < width ? b : 0.0f);
  }
}
template <int K, typename T>
__device__ __forceinline__ void store_pairs(int k, T* row, int first, int width, const Pair (&v)[4]) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) parts(v[j], f[2 * j], f[2 * j + 1]);
  if (!cut<K>(k, first, width)) {
    store8(row + first, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (first + j >= 0 && first + j < width) row[first + j] = from_float<T>(f[j]);
  }
}

// sum over a team; the two buffers take turns, so that one barrier is enough
// `name`: of the team's hardware barrier, at which all of its threads come to every sum.
template <int T>
__device__ __forceinline__ float team_sum(float a, float2 (*shared)[T / 32], int name, int& turn) {
  a = warp_sum(a);
  if (T > 32) {
    float* sums = reinterpret_cast<float*>(shared[turn]);
    if ((threadIdx.x & 31) == 0) sums[(threadIdx.x >> 5) % (T / 32)] = a;
    asm volatile("bar.sync %0, %1;" ::"r"(name), "n"(T) : "memory");
    a = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 32; ++w) a += sums[w];
    turn ^= 1;
  }
  return a;
}
// of two values
template <int T>
__device__ __forceinline__ void team_sum2(float& a, float& b, float2 (*shared)[T / 32], int name, int& turn) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (T > 32) {
    if ((threadIdx.x & 31) == 0) shared[turn][(threadIdx.x >> 5) % (T / 32)] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(name), "n"(T) : "memory");
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 32; ++w) {
      const float2 s = shared[turn][w];
      a += s.x;
      b += s.y;
    }
    turn ^= 1;
  }
}

// Bytes of the whole aligned groups among the `groups` from value `begin` on that the tensor has.
template <typename T>
__device__ __forceinline__ uint32_t row_bytes(int64_t begin, int groups, int64_t all) {
  return (uint32_t)(min((int64_t)groups * 8, all - begin) & ~(int64_t)7) * sizeof(T);
}

// A group of a row in the ring; what is not the row's reads as 0.
template <int K, typename T>
__device__ __forceinline__ void take(int k, const T* ring, int group, int first, int width, Pair (&v)[4]) {
  if (k == K - 1 && first >= width) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = pair(0.0f, 0.0f);
    return;
  }
  load_pairs(ring + group * 8, v);
  keep_pairs<K>(k, v, first, width);
}

// What the two kernels do alike: a team's rows come through its ring one after the other.  X, Y: what a row has of each type
// (Y only in the backward pass).
template <typename X, typename Y, bool kBoth>
struct Rows {
  const X* x;
  const Y* dy;
  unsigned char* shared;  // the block's dynamic shared memory
  uint32_t ring;          // where in it
  uint64_t* bars;
  int64_t row, step, rows, width, all;  // `row`: the one that is worked on
  int shift, groups, stages, stage_bytes, x_bytes;
  int at;  // stage of `row`
  uint32_t phase;
  bool gave_up;

  __device__ __forceinline__ int64_t begin_of(int64_t r) const { return r * width - shift; }
  __device__ __forceinline__ void ask(int64_t r, int stage) {  // by one thread
    unsigned char* to = shared + ring + stage * stage_bytes;
    const int64_t begin = begin_of(r);
    const uint32_t bytes = row_bytes<X>(begin, groups, all) + (kBoth ? row_bytes<Y>(begin, groups, all) : 0);
    if (begin + groups * 8 > all) {  // the rest of the last group, before the barrier hears of the row
      const int64_t whole = (all - begin) & ~(int64_t)7;
      for (int64_t i = whole; i < all - begin; ++i) {
        reinterpret_cast<X*>(to)[i] = x[begin + i];
        if (kBoth) reinterpret_cast<Y*>(to + x_bytes)[i] = dy[begin + i];
      }
    }
    mbar_expect_tx(&bars[stage], bytes);
    const uint32_t count = row_bytes<X>(begin, groups, all);
    if (count) {
      bulk_load(to, x + begin, count, &bars[stage]);
      if (kBoth) bulk_load(to + x_bytes, dy + begin, row_bytes<Y>(begin, groups, all), &bars[stage]);
    }
  }
  // the first rows; by one thread
  __device__ __forceinline__ void start() {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&bars[s], 1);
    }
    fence_mbar_init();
    for (int s = 0; s < stages - 1 && row + s * step < rows; ++s) ask(row + s * step, s);
  }
  // Once all of the team are done with the row before this one: its place in the ring takes the next row to be asked for.
  __device__ __forceinline__ void ask_next() {
    const int64_t r = row + (int64_t)(stages - 1) * step;
    if (r < rows) ask(r, at == 0 ? stages - 1 : at - 1);
  }
  __device__ __forceinline__ uint32_t wait() {  // where the row is
    // after a wait that ran out, the others (which copies may still be on their way for) are short; the sums are then wrong,
    // and the status says so
    if (!mbar_wait_bounded(&bars[at], phase, gave_up ? 1000ull * 1000 : 2000ull * 1000 * 1000)) {
      gave_up = true;
      atomicMax(&g_norm_status, 3u);
    }
    return ring + at * stage_bytes;
  }
  __device__ __forceinline__ void next() {
    row += step;
    if (++at == stages) {
      at = 0;
      phase ^= 1;
    }
  }
};

template <typename X, typename Y, bool kBoth, int T, int K>
__device__ __forceinline__ Rows<X, Y, kBoth> rows_of(const NormParams& p, unsigned char* shared, int rings, uint64_t* bars) {
  using G = Block<T, K, kBoth>;
  Rows<X, Y, kBoth> q;
  const int place = blockIdx.x % p.period;  // rows place, place + period, ... are shared out among the blocks of this place
  const int mine = threadIdx.x / T;
  q.x = static_cast<const X*>(p.x);
  q.dy = static_cast<const Y*>(p.dy);
  q.shared = shared;
  q.ring = rings + mine * p.stages * p.stage_bytes;
  q.bars = bars + mine * kMostStages;
  q.row = place + ((int64_t)(blockIdx.x / p.period) * G::kTeams + mine) * p.period;
  q.step = (int64_t)(gridDim.x / p.period) * G::kTeams * p.period;
  q.rows = p.rows;
  q.width = p.width;
  q.all = p.rows * p.width;
  q.shift = (int)(place * p.width & 7);
  q.groups = (int)((p.width + q.shift + 7) / 8);
  q.stages = p.stages;
  q.stage_bytes = p.stage_bytes;
  q.x_bytes = p.x_bytes;
  q.at = 0;
  q.phase = 0;
  q.gave_up = false;
  return q;
}

// T threads a row, K groups of eight a thread
template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(Block<T, K, false>::kThreads, 1) hc_norm_kernel(const __grid_constant__ NormParams p) {
  using G = Block<T, K, false>;
  __shared__ float2 shared[G::kTeams][2][T / 32];
  __shared__ uint64_t bars[G::kTeams * kMostStages];
  extern __shared__ __align__(16) float params[];  // w and b by place: [2][K * T * 8]; the rings
  const int lane = threadIdx.x % T, team = threadIdx.x / T;
  auto q = rows_of<X, Y, false, T, K>(p, reinterpret_cast<unsigned char*>(params), 2 * K * T * 32, bars);
  if (lane == 0) q.start();
#pragma unroll 4
  for (int i = threadIdx.x; i < K * T * 8; i += G::kThreads) {
    const int64_t c = i - q.shift;
    const bool in = c >= 0 && c < p.width;
    params[param_place<K * T * 8>(i)] = !in ? 0.0f : p.weight ? param_at(p.weight, p.param_type, c) : 1.0f;
    params[K * T * 8 + param_place<K * T * 8>(i)] = p.bias && in ? param_at(p.bias, p.param_type, c) : 0.0f;
  }
  __syncthreads();
  const float inv = 1.0f / (float)p.width;
  const int width = (int)p.width;
  int turn = 0;
  for (; q.row < q.rows; q.next()) {
    const X* x = reinterpret_cast<const X*>(reinterpret_cast<const unsigned char*>(params) + q.wait());
    Pair v[K][4], sum = pair(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      take<K>(k, x, k * T + lane, (k * T + lane) * 8 - q.shift, width, v[k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = sum + v[k][j];
    }
    const float mean = team_sum<T>(both(sum), shared[team], team + 1, turn) * inv;
    if (lane == 0) q.ask_next();
    const Pair minus = pair(-mean, -mean);
    Pair squares = pair(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = v[k][j] + minus;
      keep_pairs<K>(k, v[k], (k * T + lane) * 8 - q.shift, width);
#pragma unroll
      for (int j = 0; j < 4; ++j) squares = fma2(v[k][j], v[k][j], squares);
    }
    const float rstd = rsqrtf(fmaf(team_sum<T>(both(squares), shared[team], team + 1, turn), inv, p.eps));
    const Pair scale = pair(rstd, rstd);
    Y* y = static_cast<Y*>(p.out) + q.row * p.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = (k * T + lane) * 8 - q.shift;
      if (k == K - 1 && first >= width) continue;
      Pair w[4], b[4];
      load_params<K * T * 8>(params, k * T + lane, w);
      load_params<K * T * 8>(params + K * T * 8, k * T + lane, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = fma2(v[k][j] * scale, w[j], b[j]);
      store_pairs<K>(k, y, first, width, b);
    }
    if (p.stats && lane == 0) reinterpret_cast<float2*>(p.stats)[q.row] = make_float2(mean, rstd);
  }
}

template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(Block<T, K, true>::kThreads, 1) hc_norm_backward_kernel(const __grid_constant__ NormParams p) {
  using G = Block<T, K, true>;
  __shared__ float2 shared[G::kTeams][2][T / 32];
  __shared__ uint64_t bars[G::kTeams * kMostStages];
  extern __shared__ __align__(16) float params[];  // w by place: [K * T * 8]; the rings, whose place the sums [2][K * T * 8] take at last
  const int lane = threadIdx.x % T, team = threadIdx.x / T;
  auto q = rows_of<X, Y, true, T, K>(p, reinterpret_cast<unsigned char*>(params), K * T * 32, bars);
  if (lane == 0) q.start();
  Pair dw[K][4], db[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[k][j] = db[k][j] = pair(0.0f, 0.0f);
#pragma unroll 4
  for (int i = threadIdx.x; i < K * T * 8; i += G::kThreads) {
    const int64_t c = i - q.shift;
    params[param_place<K * T * 8>(i)] = c < 0 || c >= p.width ? 0.0f : p.weight ? param_at(p.weight, p.param_type, c) : 1.0f;
  }
  __syncthreads();
  const float inv = 1.0f / (float)p.width;
  const int width = (int)p.width;
  int turn = 0;
  float2 st = q.row < q.rows ? reinterpret_cast<const float2*>(p.stats)[q.row] : make_float2(0.0f, 0.0f);
  for (; q.row < q.rows; q.next()) {
    const float2 next_st = q.row + q.step < q.rows ? reinterpret_cast<const float2*>(p.stats)[q.row + q.step] : st;
    const X* x = reinterpret_cast<const X*>(reinterpret_cast<const unsigned char*>(params) + q.wait());
    const Y* dy = reinterpret_cast<const Y*>(reinterpret_cast<const unsigned char*>(x) + q.x_bytes);
    const Pair minus = pair(-st.x, -st.x), scale = pair(st.y, st.y);
    // outside the row dy and w are 0, and nothing that is not a number there reaches a sum of other columns
    Pair a2 = pair(0.0f, 0.0f), b2 = a2;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = (k * T + lane) * 8 - q.shift;
      Pair h[4], g[4], w[4];
      take<K>(k, x, k * T + lane, first, width, h);
      take<K>(k, dy, k * T + lane, first, width, g);
      load_params<K * T * 8>(params, k * T + lane, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = (h[j] + minus) * scale;
        dw[k][j] = fma2(g[j], h[j], dw[k][j]);
        db[k][j] = db[k][j] + g[j];
        g[j] = g[j] * w[j];
        a2 = a2 + g[j];
        b2 = fma2(g[j], h[j], b2);
      }
    }
    float a = both(a2), b = both(b2);
    team_sum2<T>(a, b, shared[team], team + 1, turn);
    if (lane == 0) q.ask_next();
    if (p.out) {
      // dx = rstd (w dy - a - h b) = rstd w dy + c0 + (x - mean) c1
      const float c0 = -a * inv * st.y, c1 = -b * inv * st.y * st.y;
      const Pair add = pair(c0, c0), slope = pair(c1, c1);
      X* dx = static_cast<X*>(p.out) + q.row * p.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int first = (k * T + lane) * 8 - q.shift;
        if (k == K - 1 && first >= width) continue;
        Pair h[4], g[4], w[4];
        load_pairs(x + (k * T + lane) * 8, h);
        load_pairs(dy + (k * T + lane) * 8, g);
        load_params<K * T * 8>(params, k * T + lane, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = fma2(g[j] * w[j], scale, fma2(h[j] + minus, slope, add));
        store_pairs<K>(k, dx, first, width, g);
      }
    }
    st = next_st;
  }
  if (!p.partial) return;
  // the block's teams one after the other: a fixed order
  float* sums = params + K * T * 8;
  float* mine = p.partial + (int64_t)blockIdx.x * 2 * p.width;
  for (int t = 0; t < G::kTeams; ++t) {
    __syncthreads();
    if (team != t) continue;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float w0, w1, b0, b1;
        parts(dw[k][j], w0, w1);
        parts(db[k][j], b0, b1);
        const int at = (k * 8 + 2 * j) * T + lane;  // neighbours of a warp lie next to each other
        float* to[4] = {sums + at, sums + at + T, sums + K * T * 8 + at, sums + K * T * 8 + at + T};
        *to[0] = t ? *to[0] + w0 : w0;
        *to[1] = t ? *to[1] + w1 : w1;
        *to[2] = t ? *to[2] + b0 : b0;
        *to[3] = t ? *to[3] + b1 : b1;
      }
  }
  __syncthreads();
  for (int64_t c = threadIdx.x; c < p.width; c += G::kThreads) {
    const int i = (int)c + q.shift, group = i / 8, at = (group / T * 8 + i % 8) * T + group % T;
    mine[c] = sums[at];
    mine[p.width + c] = sums[K * T * 8 + at];
  }
}

// Rows too long for the registers of a block: three passes over the row, of which the later ones find it in L2.
constexpr int kLong = 1024;
template <typename X, typename Y>
__global__ void __launch_bounds__(kLong) hc_norm_long_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[kLong / 32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    Y* y = static_cast<Y*>(p.out) + row * p.width;
    const int64_t start = -(int64_t)(row * p.width & 7) + threadIdx.x * 8;
    float v[8], sum = 0.0f, squares = 0.0f, none = 0.0f;
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    }
    group_sum2<kLong>(sum, none, shared);
    const float mean = sum * inv;
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = f + j >= 0 && f + j < p.width ? v[j] - mean : 0.0f;
        squares = fmaf(c, c, squares);
      }
    }
    none = 0.0f;
    group_sum2<kLong>(squares, none, shared);
    const float rstd = 1.0f / sqrtf(fmaf(squares, inv, p.eps));
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = f + j;
        const bool in = c >= 0 && c < p.width;
        v[j] = fmaf((v[j] - mean) * rstd, p.weight && in ? param_at(p.weight, p.param_type, c) : 1.0f,
                    p.bias && in ? param_at(p.bias, p.param_type, c) : 0.0f);
      }
      store_group(y, f, p.width, v);
    }
    if (p.stats && threadIdx.x == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(mean, rstd);
  }
}

template <typename X, typename Y>
__global__ void __launch_bounds__(kLong) hc_norm_long_dx_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[kLong / 32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    const Y* dy = static_cast<const Y*>(p.dy) + row * p.width;
    X* dx = static_cast<X*>(p.out) + row * p.width;
    const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
    const int64_t start = -(int64_t)(row * p.width & 7) + threadIdx.x * 8;
    float v[8], g[8], a = 0.0f, b = 0.0f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t f = start; f < p.width; f += kLong * 8) {
        load_group(x, f, p.width, v);
        load_group(dy, f, p.width, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t c = f + j;
          v[j] = (v[j] - st.x) * st.y;
          if (p.weight && c >= 0 && c < p.width) g[j] *= param_at(p.weight, p.param_type, c);
          if (pass == 0) {
            a += g[j];
            b = fmaf(g[j], v[j], b);
          } else {
            g[j] = st.y * (fmaf(-v[j], b, g[j]) - a);
          }
        }
        if (pass == 1) store_group(dx, f, p.width, g);
      }
      if (pass == 0) {
        group_sum2<kLong>(a, b, shared);
        a *= inv;
        b *= inv;
      }
    }
  }
}

// column sums of a share of the rows (blockIdx.y), one thread a column
template <typename X, typename Y>
__global__ void __launch_bounds__(256) hc_norm_long_sums_kernel(const __grid_constant__ NormParams p) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
    const float g = to_float(static_cast<const Y*>(p.dy)[row * p.width + c]);
    dw = fmaf(g, (to_float(static_cast<const X*>(p.x)[row * p.width + c]) - st.x) * st.y, dw);
    db += g;
  }
  float* mine = p.partial + (int64_t)blockIdx.y * 2 * p.width;
  mine[c] = dw;
  mine[p.width + c] = db;
}

// adds up the partial sums of `n` blocks: 32 columns a block of 32 x 32 threads, always in the same order
__global__ void __launch_bounds__(1024) hc_norm_finish_kernel(const float* partial, int n, int64_t width, void* dweight,
                                                               void* dbias, int param_type) {
  __shared__ float sums[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < width)
    for (int b = threadIdx.y; b < n; b += 32) s += partial[((int64_t)b * 2 + blockIdx.y) * width + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(sums[threadIdx.x][threadIdx.y]);
  if (threadIdx.x == 0) {
    const int64_t at = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (at < width) param_put(blockIdx.y ? dbias : dweight, param_type, at, s);
  }
}

}  // namespace dev

namespace {

constexpr int64_t kLongestInRegisters = 8192;

// Threads and groups of eight a thread for rows of `width` values (with one group more where rows begin anywhere).  What a row
// costs a warp besides its values, some 200 instructions, is shared by as few warps as the registers allow: up to five groups a
// thread (6001 x 5003 bf16: with 256 threads a row and three groups 43 us forward and 55 us back, with 128 and five 37 and 54, although
// the backward pass then has 36 to 112 bytes more to a thread than its 128 registers hold).
// Forward a warp alone takes rows of up to three groups a thread, with no barrier in its sums (8192 x 768: 12.9 us, 17.7 with 128
// threads); back, where it would have 24 column sums a thread and rings for 16 teams, it does not (24.1 us, 20.1).  Long rows
// of wide types have fewer teams, for whose rings there is room.
struct Shape {
  int threads, groups;
};
constexpr int block_threads(bool backward, int groups) { return backward || groups > 3 ? 512 : 1024; }
int ring_stages(bool backward, Shape s, size_t width, size_t bytes) {
  const size_t groups = (width + 7) / 8 + (width % 8 ? 1 : 0), params = (size_t)s.groups * s.threads * 32 * (backward ? 1 : 2);
  return (int)((dev::kNormSmem - params) / (block_threads(backward, s.groups) / s.threads) / (groups * 8 * bytes));
}
// bytes: of a value of x, and of dy in the backward pass
Shape shape_of(bool backward, size_t width, size_t bytes) {
  const int need = (int)((width + 7) / 8) + (width % 8 ? 1 : 0);
  if (!backward && need <= 96) return {32, (need + 31) / 32};
  if (need <= 128) return {need <= 32 ? 32 : need <= 64 ? 64 : 128, 1};
  const Shape one = {128, (need + 127) / 128}, two = {256, (need + 255) / 256};
  if (need <= 640 && ring_stages(backward, one, width, bytes) >= 2) return one;
  return ring_stages(backward, two, width, bytes) >= 2 ? two : Shape{512, 2};
}
int period_of(size_t width) { return width % 8 == 0 ? 1 : width % 4 == 0 ? 2 : width % 2 == 0 ? 4 : 8; }
bool in_registers(size_t width) { return width <= kLongestInRegisters - (width % 8 ? 8 : 0); }

// Blocks: one an SM, a whole number of them for each place of an aligned group, and no more than have a row for a team
int norm_blocks(size_t rows, size_t width, int teams) {
  const int sms = device_info().sms > 0 ? device_info().sms : 1;
  if (!in_registers(width)) return (int)(rows < 64 ? rows : 64);
  const int period = period_of(width);
  const size_t most = (size_t)(sms < period ? period : sms / period * period);
  const size_t blocks = (rows + (size_t)teams * period - 1) / ((size_t)teams * period) * period;
  return (int)(blocks < most ? blocks : most);
}

// the rings' part of the shared memory, `other` bytes of it apart; at least `least` bytes
int plan_rings(dev::NormParams* p, size_t x_bytes, size_t y_bytes, int teams, int other, int least) {
  const size_t groups = (p->width + 7) / 8 + (p->width % 8 ? 1 : 0);
  p->x_bytes = (int)(groups * 8 * x_bytes);
  p->stage_bytes = (int)(groups * 8 * (x_bytes + y_bytes));
  int stages = (dev::kNormSmem - other) / teams / p->stage_bytes;
  if (stages > dev::kMostStages) stages = dev::kMostStages;
  p->stages = stages;
  const int rings = stages * teams * p->stage_bytes;
  return other + (rings > least ? rings : least);
}

template <typename X, typename Y, int T, int K>
cudaError_t run_forward(dev::NormParams p, cudaStream_t stream) {
  using G = dev::Block<T, K, false>;
  const int smem = plan_rings(&p, sizeof(X), 0, G::kTeams, 2 * K * T * 8 * 4, 0);
  if (p.stages < 2) return cudaErrorInvalidConfiguration;
  static unsigned long long allowed = 0;
  const cudaError_t e = allow_smem(dev::hc_norm_kernel<X, Y, T, K>, dev::kNormSmem, &allowed);
  if (e != cudaSuccess) return e;
  dev::hc_norm_kernel<X, Y, T, K><<<norm_blocks(p.rows, p.width, G::kTeams), G::kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}
template <typename X, typename Y, int T, int K>
cudaError_t run_backward(dev::NormParams p, int* blocks, cudaStream_t stream) {
  using G = dev::Block<T, K, true>;
  const int smem = plan_rings(&p, sizeof(X), sizeof(Y), G::kTeams, K * T * 8 * 4, 2 * K * T * 8 * 4);
  if (p.stages < 2) return cudaErrorInvalidConfiguration;
  static unsigned long long allowed = 0;
  const cudaError_t e = allow_smem(dev::hc_norm_backward_kernel<X, Y, T, K>, dev::kNormSmem, &allowed);
  if (e != cudaSuccess) return e;
  *blocks = norm_blocks(p.rows, p.width, G::kTeams);
  dev::hc_norm_backward_kernel<X, Y, T, K><<<*blocks, G::kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

// f with the threads and groups as constants
template <bool kBackward, typename F>
cudaError_t by_shape(size_t width, size_t bytes, F f) {
  const Shape s = shape_of(kBackward, width, bytes);
  if (s.threads == 32) {
    if (s.groups == 1) return f.template run<32, 1>();
    if constexpr (!kBackward) return s.groups == 2 ? f.template run<32, 2>() : f.template run<32, 3>();
  }
  if constexpr (kBackward)
    if (s.threads == 64) return f.template run<64, 1>();
  if (s.threads == 128) {
    if (s.groups == 1) return f.template run<128, 1>();
    if (s.groups == 2) return f.template run<128, 2>();
    if (s.groups == 3) return f.template run<128, 3>();
    return s.groups == 4 ? f.template run<128, 4>() : f.template run<128, 5>();
  }
  if (s.threads == 256) {
    if constexpr (kBackward)
      if (s.groups == 2) return f.template run<256, 2>();
    return s.groups == 3 ? f.template run<256, 3>() : f.template run<256, 4>();
  }
  return f.template run<512, 2>();
}
template <typename X, typename Y>
struct Forward {
  const dev::NormParams& p;
  cudaStream_t stream;
  template <int T, int K>
  cudaError_t run() {
    return run_forward<X, Y, T, K>(p, stream);
  }
};
template <typename X, typename Y>
struct Backward {
  const dev::NormParams& p;
  int* blocks;
  cudaStream_t stream;
  template <int T, int K>
  cudaError_t run() {
    return run_backward<X, Y, T, K>(p, blocks, stream);
  }
};

template <typename X, typename Y>
cudaError_t forward(const dev::NormParams& p, cudaStream_t stream) {
  if (in_registers(p.width)) return by_shape<false>(p.width, sizeof(X), Forward<X, Y>{p, stream});
  dev::hc_norm_long_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
  return cudaGetLastError();
}
template <typename X, typename Y>
cudaError_t backward(const dev::NormParams& p, int* blocks, cudaStream_t stream) {
  if (in_registers(p.width)) return by_shape<true>(p.width, sizeof(X) + sizeof(Y), Backward<X, Y>{p, blocks, stream});
  *blocks = norm_blocks(p.rows, p.width, 1);
  if (p.out) dev::hc_norm_long_dx_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
  if (p.partial) dev::hc_norm_long_sums_kernel<X, Y><<<dim3((unsigned)((p.width + 255) / 256), *blocks), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename F>
cudaError_t by_types(int x, int y, F f) {
  using b = __nv_bfloat16;
  using h = __half;
  if (x == kF32) return y == kF32 ? f(float(), float()) : y == kBf16 ? f(float(), b()) : f(float(), h());
  if (x == kBf16) return y == kF32 ? f(b(), float()) : y == kBf16 ? f(b(), b()) : cudaErrorInvalidValue;
  return y == kF32 ? f(h(), float()) : y == kF16 ? f(h(), h()) : cudaErrorInvalidValue;
}

bool norm_arguments_ok(const void* x, int x_type, const void* y, int y_type, int param_type, size_t rows, size_t width) {
  if (!element_type_ok(x_type) || !element_type_ok(y_type) || !element_type_ok(param_type)) return false;
  if (x_type != kF32 && y_type != kF32 && x_type != y_type) return false;
  if (width == 0 || width > (1u << 30) || rows > (1ull << 40) || rows > (1ull << 60) / width) return false;
  return rows == 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
}

}  // namespace

int norm_status(int clear) { return take_status(dev::g_norm_status, clear); }

}  // namespace hc

extern "C" {

int hc_layer_norm(const void* x, int x_type, const void* weight, const void* bias, int param_type, void* y, int y_type,
                  float* stats, size_t rows, size_t width, float eps, hc_stream_t stream) {
  if (!hc::norm_arguments_ok(x, x_type, y, y_type, param_type, rows, width) || !(eps >= 0.0f)) return hc::kErrArgument;
  if (rows == 0) return hc::kOk;
  if (!x || !y) return hc::kErrArgument;
  const size_t param = hc::element_bytes(param_type);
  if (!hc::lies_at(weight, param) || !hc::lies_at(bias, param) || !hc::lies_at(stats, 8)) return hc::kErrArgument;
  hc::dev::NormParams p = {x, nullptr, weight, bias, y, stats, nullptr, (int64_t)rows, (int64_t)width, eps, param_type, hc::period_of(width), 0, 0, 0};
  const cudaError_t e = hc::by_types(x_type, y_type, [&](auto a, auto b) { return hc::forward<decltype(a), decltype(b)>(p, stream); });
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

size_t hc_layer_norm_backward_bytes(size_t rows, size_t width) {
  return rows && width ? (size_t)hc::norm_blocks(rows, width, 1) * 2 * width * sizeof(float) : 0;
}

int hc_layer_norm_backward(const void* dy, int y_type, const void* x, int x_type, const void* weight, int param_type,
                           const float* stats, void* dx, void* dweight, void* dbias, size_t rows, size_t width,
                           void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  if (!hc::norm_arguments_ok(x, x_type, dy, y_type, param_type, rows, width) || (!dweight != !dbias)) return hc::kErrArgument;
  const size_t param = hc::element_bytes(param_type);
  if (!hc::lies_at(dx, 16) || !hc::lies_at(weight, param) || !hc::lies_at(dweight, param) || !hc::lies_at(dbias, param) || !hc::lies_at(stats, 8) ||
      !hc::lies_at(scratch, 256))
    return hc::kErrArgument;
  if (rows == 0) {
    if (!dweight) return hc::kOk;
    cudaError_t e = cudaMemsetAsync(dweight, 0, width * hc::element_bytes(param_type), stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, width * hc::element_bytes(param_type), stream);
    return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
  }
  if (!x || !dy || !stats) return hc::kErrArgument;
  if (!dx && !dweight) return hc::kOk;
  int blocks = 0;  // at most as many as with a row a block
  if (dweight && (!scratch || scratch_bytes < hc_layer_norm_backward_bytes(rows, width))) return hc::kErrArgument;
  hc::dev::NormParams p = {x, dy, weight, nullptr, dx, const_cast<float*>(stats), dweight ? static_cast<float*>(scratch) : nullptr,
                           (int64_t)rows, (int64_t)width, 0.0f, param_type, hc::period_of(width), 0, 0, 0};
  cudaError_t e = hc::by_types(x_type, y_type, [&](auto a, auto b) { return hc::backward<decltype(a), decltype(b)>(p, &blocks, stream); });
  if (e == cudaSuccess && dweight) {
    hc::dev::hc_norm_finish_kernel<<<dim3((unsigned)((width + 31) / 32), 2), dim3(32, 32), 0, stream>>>(
        p.partial, blocks, (int64_t)width, dweight, dbias, param_type);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

}  // extern "C"
