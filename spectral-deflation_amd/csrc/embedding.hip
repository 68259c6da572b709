// Embedding lookup with scaling, and its gradients by sorted tokens.
//
//   out[i, :]  = D(scale * W[id_i, :] + P[pos_i, :])
//   dW[v, :]  (+)= scale * sum over i with id_i = v of D(g)[i, :]
//   dP[t, :]  (+)= sum over i with pos_i = t of D(g)[i, :]
//
// D is dropout over the flat index i * dim + column (train_ops.h), evaluated again in the
// backward pass.  Sums are held in fp32 and taken in the order of the tokens: no atomics, the
// same gradient every time.  An id or position outside its table gives a row of NaN, and no
// gradient.
#include "train_ops.h"

namespace dmh {

struct EmbedArgs {
  const void* ids;
  const void* pos;        // positions, or null: i % seq
  const void* w;
  const void* p;          // position table, or null
  void* out;
  long long tokens, vocab, wstride, prows, pstride;
  int is64, seq, dim;
  int lanes, log_lanes;   // of a token
  float scale;
  Rng rng;
};

// Bound by the rows it reads and writes: 8192 tokens of 1280 fp32 columns with positions and
// dropout take 14.1 us, 65 MB at 4.6 TB/s, where the tables' rows are in the last-level cache from
// the call before.  In a training step they come from HBM, and it takes 25.3.
//
// A token is `lanes` (a power of two up to a wave) neighbouring lanes' work, which take eight of
// its columns each, `lanes` pieces apart: as many as leave the fewest idle at the row's end, so
// that ids, positions and row addresses are found once for several pieces and without divisions.
// The last eight columns of a row overlap those before them where the width is no multiple of
// eight (SPLIT), and are written twice with the same values; rows narrower than eight go column
// by column (NARROW).  With a division for every eight columns 27000 tokens of 1536 bf16 columns
// with dropout took 35.9 us, now 29.1.
template <class TW, class TO, bool POS, bool DROP, bool SPLIT, bool NARROW>
__global__ __launch_bounds__(256) void embed_rows(EmbedArgs a) {
  constexpr int W = NARROW ? 1 : 8, AHEAD = 2;
  const int lane = threadIdx.x & (a.lanes - 1);
  const long long step = (long long)gridDim.x * (256 >> a.log_lanes);
  const RngKey key = DROP ? rng_key(a.rng) : RngKey{};
  for (long long i = (long long)blockIdx.x * (256 >> a.log_lanes) + (threadIdx.x >> a.log_lanes);
       i < a.tokens; i += step) {
    const long long id = load_index(a.ids, a.is64, i);
    const long long t = !POS    ? 0
                        : a.pos ? load_index(a.pos, a.is64, i)
                        : a.tokens < (1LL << 32) ? (unsigned)i % (unsigned)a.seq
                                                 : i % a.seq;
    const bool ok = (unsigned long long)id < (unsigned long long)a.vocab &&
                    (!POS || (unsigned long long)t < (unsigned long long)a.prows);
    const unsigned long long row = (unsigned long long)i * a.dim;
    TO* out = (TO*)a.out + row;
    const TW* w = (const TW*)a.w + (ok ? id : 0) * a.wstride;
    const TW* p = (const TW*)a.p + (ok ? t : 0) * a.pstride;
    if (!ok) {
      for (int c = lane; c < a.dim; c += a.lanes) out[c] = (TO)__builtin_nanf("");
    } else if (NARROW) {
      for (int c = lane; c < a.dim; c += a.lanes) {
        float v = POS ? fmaf((float)w[c], a.scale, (float)p[c]) : (float)w[c] * a.scale;
        if (DROP) v = kept(keep_bits_at<true>(a.rng, key, row + c), 0, v * a.rng.scale);
        out[c] = (TO)v;
      }
    } else {
      for (int c0 = lane * W; c0 < a.dim; c0 += AHEAD * W * a.lanes) {
        Raw8<TW> x[AHEAD], q[AHEAD];
        int c[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          c[k] = c0 + k * W * a.lanes;
          // beyond the row: the piece before again
          c[k] = c[k] >= a.dim ? c0 : c[k];
          c[k] = SPLIT && c[k] + 8 > a.dim ? a.dim - 8 : c[k];
          x[k].load(w + c[k]);
          if (POS) q[k].load(p + c[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (k && c0 + k * W * a.lanes >= a.dim) break;
          const uint32_t bits = DROP ? keep_bits_at<SPLIT>(a.rng, key, row + c[k]) : 0;
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = POS ? fmaf(x[k][j], a.scale, q[k][j]) : x[k][j] * a.scale;
            if (DROP) v[j] = kept(bits, j, v[j] * a.rng.scale);
          }
          store8(out + c[k], v);
        }
      }
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------
// Bound by its bytes: the dense gradient that is written, most of it zeros (257 MB of the 304 that
// 8192 tokens of GPT-2 large move), and the rows of the gradient, once a table.
//
// A table's gradient is a job: its tokens are put in the order of (id, index), the sorted
// tokens are cut into chunks, and a wave adds up the rows of one chunk and 512 columns, id by
// id.  What lies in one chunk goes straight to the table; an id that reaches over a chunk's end
// leaves its parts in the workspace, which a last launch joins.  So the work is even however
// the ids are distributed, every sum is taken in one order, and there are no atomics on values.
// Rows that no token names are cleared by the workgroups of the same launch that find no id of
// theirs in the sorted list.
//
// Implicit positions (i % seq) need no sort: sorted place s is token (s % batch) seq + s / batch.
struct GradJob {
  const void* ids;     // null: implicit positions
  void* out;
  int* keys;           // sorted ids
  int* order;          // their tokens
  int* keys2;          // the radix sort's other buffers
  int* order2;
  int* hist;
  float* part;         // two rows of `dimp` a chunk: [0] of an id that began before the chunk,
                       // [1] of one that begins in it and goes on
  long long padding;
  int rows;
  int accumulate;
  float scale;
  int chunks;          // of sorted tokens
  int reduce_groups, fill_groups;   // workgroups of embed_grad
  int spans;           // some id may reach over a chunk's end
};
struct GradArgs {
  GradJob job[2];      // the token table's and the position table's
  const void* g;
  long long gstride;
  int is64, tokens, seq, batch, dim, dimp, ctiles, lanes;   // a wave: `lanes` x 8 columns
  int small;           // embed_grad_small's
  Rng rng;
};

// Ids that take no gradient (padding, outside the table) sort behind all others, as `rows`.
__device__ __forceinline__ int sort_key(const GradJob& j, long long id) {
  return (unsigned long long)id < (unsigned long long)j.rows && id != j.padding ? (int)id : j.rows;
}

// Few tokens: the place of a token is the number of tokens before it in the order of (id,
// index), counted against all of them.  A workgroup places 32 tokens; the keys lie in LDS, and
// lane pairs of its waves take a share of them each.  8192 tokens take 9.6 us in one launch,
// where the radix sort's four take 20; 13662 tokens are no faster this way than that.
constexpr int RANK_MAX = 8192, RANK_TOKENS = 32, RANK_THREADS = 512;

__global__ __launch_bounds__(RANK_THREADS) void embed_rank(GradArgs a) {
  __shared__ __attribute__((aligned(16))) int keys[RANK_MAX];
  __shared__ int count[RANK_TOKENS];
  const GradJob& j = a.job[blockIdx.y + !a.job[0].ids];
  constexpr int SHARES = RANK_THREADS / RANK_TOKENS, ROUNDS = RANK_MAX / RANK_THREADS;
  const int n = a.tokens, i0 = blockIdx.x * RANK_TOKENS;
  // padded to a multiple of 16 keys a share (n <= RANK_MAX, a multiple of 16 SHARES)
  const int len = ((n + SHARES - 1) / SHARES + 15) & ~15;
  {
    // all loads on their way before the first is used
    long long id[ROUNDS];
    if (a.is64) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int s = r * RANK_THREADS + threadIdx.x;
        id[r] = ((const long long*)j.ids)[s < n ? s : 0];
      }
    } else {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int s = r * RANK_THREADS + threadIdx.x;
        id[r] = ((const int*)j.ids)[s < n ? s : 0];
      }
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int s = r * RANK_THREADS + threadIdx.x;
      keys[s] = s < n ? sort_key(j, id[r]) : 0x7FFFFFFF;   // before none
    }
  }
  if (threadIdx.x < RANK_TOKENS) count[threadIdx.x] = 0;
  __syncthreads();
  const int i = i0 + (threadIdx.x & (RANK_TOKENS - 1));
  const int share = threadIdx.x / RANK_TOKENS;
  const int mine = i < n ? keys[i] : 0;
  const int s0 = share * len;
  int before = 0;
  // equal keys count if their token is before this one: all those of 16 keys before this
  // workgroup's tokens, none of those behind them
#pragma unroll 2
  for (int s = s0; s < s0 + len; s += 16) {
    const int t = mine + (s < i0);
    int c = 0;
#pragma unroll
    for (int q = 0; q < 16; q += 4) {
      const int4 k = *(const int4*)(keys + s + q);
      c += (k.x < t) + (k.y < t) + (k.z < t) + (k.w < t);
    }
    before += c;
  }
  if (share < 2)   // the workgroup's own tokens: half of them in each share
    for (int q = 0; q < RANK_TOKENS / 2; ++q) {
      const int s = i0 + share * (RANK_TOKENS / 2) + q;
      before += s < i && keys[s] == mine;
    }
  atomicAdd(&count[threadIdx.x & (RANK_TOKENS - 1)], before);
  __syncthreads();
  if (share == 0 && i < n) {
    const int at = count[threadIdx.x];
    j.keys[at] = mine;
    j.order[at] = i;
  }
}

// Many tokens: a stable radix sort, eight bits a pass from the lowest.  At most 256 workgroups
// take an equal run of the list each: one launch counts the run's digits, the next adds up the
// counts of the runs before it and moves the run's keys, in order.  32768 tokens of 16-bit ids:
// 4.7 and 6.4 us a pass, latency all of it.
constexpr int RADIX_RUNS = 256, RADIX_ROUND = 1024;

__device__ __forceinline__ int radix_run(int tokens, int runs) {
  const int len = (tokens + runs - 1) / runs;
  return (len + RADIX_ROUND - 1) / RADIX_ROUND * RADIX_ROUND;
}

__global__ __launch_bounds__(256) void radix_count(GradArgs a, int pass, int runs, int parity) {
  __shared__ int hist[256];
  const GradJob& j = a.job[blockIdx.y + !a.job[0].ids];
  const int* src = parity ? j.keys2 : j.keys;   // pass 0 reads the ids
  hist[threadIdx.x] = 0;
  __syncthreads();
  const long long len = radix_run(a.tokens, runs), i0 = blockIdx.x * len;
  const long long i1 = i0 + len < a.tokens ? i0 + len : a.tokens;
  for (long long i = i0 + threadIdx.x; i < i1; i += 256) {
    const int k = pass ? src[i] : sort_key(j, load_index(j.ids, a.is64, i));
    atomicAdd(&hist[(unsigned)k >> (8 * pass) & 255], 1);
  }
  __syncthreads();
  j.hist[blockIdx.x * 256 + threadIdx.x] = hist[threadIdx.x];
}

// A pass of parity 1 reads keys2 / order2 and writes keys / order, the last pass among them;
// the others the other way.
__global__ __launch_bounds__(256) void radix_move(GradArgs a, int pass, int runs, int parity) {
  __shared__ int base[256];       // next place of each digit
  __shared__ int cnt[4][256];     // keys of each digit in each wave's part of a round
  __shared__ int wsum[4];
  const GradJob& j = a.job[blockIdx.y + !a.job[0].ids];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int* ksrc = parity ? j.keys2 : j.keys;
  const int* osrc = parity ? j.order2 : j.order;
  int* kdst = parity ? j.keys : j.keys2;
  int* odst = parity ? j.order : j.order2;
  {
    int total = 0, mine = 0;
#pragma unroll 8
    for (int r = 0; r < runs; ++r) {
      const int c = j.hist[r * 256 + threadIdx.x];
      total += c;
      if (r < (int)blockIdx.x) mine += c;
    }
    int scan = total;             // over the digits, then without itself
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(scan, d);
      if (lane >= d) scan += up;
    }
    if (lane == 63) wsum[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) scan += wsum[w];
    base[threadIdx.x] = scan - total + mine;
  }
  const long long len = radix_run(a.tokens, runs), r0 = blockIdx.x * len;
  const long long r1 = r0 + len < a.tokens ? r0 + len : a.tokens;
  for (long long i0 = r0; i0 < r1; i0 += RADIX_ROUND) {
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w][threadIdx.x] = 0;
    __syncthreads();
    int key[4], tok[4], rank[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long i = i0 + wave * 256 + q * 64 + lane;
      key[q] = i >= r1 ? 0 : pass ? ksrc[i] : sort_key(j, load_index(j.ids, a.is64, i));
      tok[q] = i >= r1 ? 0 : pass ? osrc[i] : (int)i;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool in = i0 + wave * 256 + q * 64 + lane < r1;
      const int d = (unsigned)key[q] >> (8 * pass) & 255;
      unsigned long long same = __ballot(in);   // lanes with a key of this digit
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const unsigned long long set = __ballot(d >> bit & 1);
        same &= d >> bit & 1 ? set : ~set;
      }
      const int below = __popcll(same & ((1ull << lane) - 1));
      // a wave's LDS accesses are in order; the barriers keep the compiler from moving them
      const int before = in ? cnt[wave][d] : 0;
      __builtin_amdgcn_wave_barrier();
      if (in && below == 0) cnt[wave][d] = before + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      rank[q] = before + below;
    }
    __syncthreads();
    int at = base[threadIdx.x];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = at;
      at += c;
    }
    base[threadIdx.x] = at;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (i0 + wave * 256 + q * 64 + lane < r1) {
        const int to = cnt[wave][(unsigned)key[q] >> (8 * pass) & 255] + rank[q];
        kdst[to] = key[q];
        odst[to] = tok[q];
      }
    }
    __syncthreads();
  }
}

// sorted ids and their tokens
__device__ __forceinline__ int key_at(const GradArgs& a, const GradJob& j, int s) {
  return j.ids ? j.keys[s] : s / a.batch;
}
__device__ __forceinline__ int token_at(const GradArgs& a, const GradJob& j, int s) {
  return j.ids ? j.order[s] : (s % a.batch) * a.seq + s / a.batch;
}

// First of the sorted keys lo .. hi - 1 that is not below v (hi if none): by one lane, and by a
// wave together, 64 probes a step.
__device__ __forceinline__ int first_at(const int* keys, int lo, int hi, int v) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int wave_first_at(const int* keys, int hi, int v) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (lo < hi) {
    const int step = (hi - lo + 63) >> 6;
    const int p = lo + lane * step;          // lane's share: p .. p + step - 1
    const int last = p + step - 1 < hi ? p + step - 1 : hi - 1;
    const int full = __popcll(__ballot(p < hi && keys[p < hi ? last : lo] < v));
    lo = lo + full * step < hi ? lo + full * step : hi;
    hi = lo + step - 1 < hi ? lo + step - 1 : hi;
  }
  return lo;
}

// The scaled sum of one id into eight columns of its row.  The last eight columns of a width that is
// no multiple of eight begin inside the piece before them, and the two lanes, which lie in one
// wave (grad_lanes), write what they share with the same values.  Where sums are added both
// have to read it before either writes: the wave's loads stand before the fence, its stores
// behind it.  (With the shared columns left to one lane, by stores one by one, 8192 tokens
// added to 50257 rows took 52 us instead of 47 for 1283 columns and, for the branch alone, 46
// instead of 44 for 1280.)
template <class TO>
__device__ __forceinline__ void put_row(const GradArgs& a, const GradJob& j, int row, int c,
                                        const float (&sum)[8]) {
  TO* o = (TO*)j.out + (long long)row * a.dim + c;
  float v[8] = {};
  if (j.accumulate) {
    load8(o, v);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = fmaf(sum[k], j.scale, v[k]);
  store8(o, v);
}

// Sorted tokens a chunk: 16 leave twice the parts to join (32768 tokens 115 us instead of 101),
// 64 half the waves (8192 tokens 81 us instead of 68).
constexpr int CHUNK = 32;
constexpr int FILL_ROWS = 64;   // table rows a workgroup clears
// Rows of the gradient that a wave loads ahead, without a branch between them: with loads that
// wait for one another the launch of 8192 tokens took 60 us instead of 51, eight rows ahead take
// 3 us more.
constexpr int IN_FLIGHT = 16;

// The rows of a table that no token names: 7.5 TB/s by itself.  Clearing a part of the table in
// the sort's launches instead, which leave the memory idle, gained nothing; nor did the position
// table's sums there, which then no longer share the gradient's rows with the token table's.
template <class TO>
__device__ void clear_rows(const GradArgs& a, const GradJob& j, int group) {
  __shared__ int bound[2];
  __shared__ unsigned long long named;
  const int v0 = group * FILL_ROWS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (j.ids && wave < 2) {   // the places of this workgroup's rows in the sorted keys
    const int s = wave_first_at(j.keys, a.tokens, v0 + wave * FILL_ROWS);
    if (lane == 0) bound[wave] = s;
  }
  __syncthreads();
  if (wave == 0) {
    const int v = v0 + lane;
    bool hit = v >= j.rows;
    if (!hit && j.ids) {
      const int s = first_at(j.keys, bound[0], bound[1], v);
      hit = s < bound[1] && j.keys[s] == v;
    } else if (!hit) {
      hit = a.tokens > 0 && v < a.seq;
    }
    const unsigned long long m = __ballot(hit);
    if (lane == 0) named = m;
  }
  __syncthreads();
  const unsigned long long m = named;
  if (a.dim < 8) {   // rows shorter than a piece: all of them together
    const int count = (j.rows - v0 < FILL_ROWS ? j.rows - v0 : FILL_ROWS) * a.dim;
    TO* o = (TO*)j.out + (long long)v0 * a.dim;
    for (int e = threadIdx.x; e < count; e += 256)
      if (!(m >> (e / a.dim) & 1)) o[e] = (TO)0.f;
    return;
  }
  constexpr int N = Piece<TO>::N;
  const typename Piece<TO>::type zero = {};
  const int whole = a.dim / N;
  for (int r = wave; r < FILL_ROWS; r += 4) {
    if (m >> r & 1) continue;
    TO* o = (TO*)j.out + (long long)(v0 + r) * a.dim;
    for (int p = lane; p < whole; p += 64) *(typename Piece<TO>::type*)(o + p * N) = zero;
    if (lane < a.dim - whole * N) o[whole * N + lane] = (TO)0.f;
  }
}

// Sums and cleared rows in one launch: 51 us for 8192 tokens of 1280 fp32 columns into 50257 and
// 1024 rows with dropout (346 MB with the gradient's second reading: 6.8 TB/s), 68 us for 32768
// bf16 ones (431 MB, 6.3 TB/s).
//
// A lane has eight columns.  Where the width is no multiple of eight, the last lane of a row takes
// its last eight columns, some of them its neighbour's too (put_row).
template <class TG, class TO, bool DROP>
__global__ __launch_bounds__(256) void embed_grad(GradArgs a) {
  // the sums first: their latency is under the writes of the rows cleared behind them
  const int sums = a.job[0].reduce_groups + a.job[1].reduce_groups;
  int b = blockIdx.x;
  if (b >= sums) {
    b -= sums;
    const int second = b >= a.job[0].fill_groups;
    clear_rows<TO>(a, a.job[second], second ? b - a.job[0].fill_groups : b);
    return;
  }
  const int jn = b >= a.job[0].reduce_groups;
  const GradJob& j = a.job[jn];
  if (jn) b -= a.job[0].reduce_groups;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(b * 4 + (int)(threadIdx.x >> 6));
  const int chunk = w / a.ctiles;
  if (chunk >= j.chunks) return;
  int c = ((w - chunk * a.ctiles) * a.lanes + lane) * 8;
  const bool mine = lane < a.lanes && c < a.dim;
  c = mine && c + 8 <= a.dim ? c : a.dim - 8;   // lanes without columns read, and write nothing
  const int s0 = chunk * CHUNK, count = a.tokens - s0 < CHUNK ? a.tokens - s0 : CHUNK;
  // lane l has the chunk's entry l; behind the last one, that one again
  const int sl = s0 + (lane < count ? lane : count - 1);
  const int key = key_at(a, j, sl), tok = token_at(a, j, sl);
  const int before = s0 ? key_at(a, j, s0 - 1) : -1;
  const int after = s0 + count < a.tokens ? key_at(a, j, s0 + count) : -1;
  const RngKey rk = DROP ? rng_key(a.rng) : RngKey{};
  const TG* g = (const TG*)a.g + c;
  float* part = j.part + (long long)chunk * 2 * a.dimp + c;
  float sum[8] = {};
  int cur = __builtin_amdgcn_readlane(key, 0);
  bool began_here = cur != before;
  for (int e0 = 0; e0 < count; e0 += IN_FLIGHT) {
    Raw8<TG> x[IN_FLIGHT];
#pragma unroll
    for (int q = 0; q < IN_FLIGHT; ++q)
      x[q].load(g + (long long)__builtin_amdgcn_readlane(tok, e0 + q) * a.gstride);
    // the masks of four rows to a word, while the rows are on their way
    uint32_t bits[IN_FLIGHT / 4];
    if (DROP) {
#pragma unroll
      for (int q4 = 0; q4 < IN_FLIGHT / 4; ++q4) {
        bits[q4] = 0;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const unsigned long long e =
              (unsigned long long)__builtin_amdgcn_readlane(tok, e0 + q4 * 4 + q) * a.dim + c;
          bits[q4] |= (a.dim & 7 ? keep_bits_at<true>(a.rng, rk, e)
                                 : keep_bits_at<false>(a.rng, rk, e)) << (4 * q);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < IN_FLIGHT; ++q) {
      if (e0 + q >= count) break;
      const int k = __builtin_amdgcn_readlane(key, e0 + q);
      if (k != cur) {
        if (mine) {
          if (began_here) put_row<TO>(a, j, cur, c, sum); else store8(part, sum);
        }
        cur = k;
        began_here = true;
#pragma unroll
        for (int z = 0; z < 8; ++z) sum[z] = 0.f;
      }
      if (k >= j.rows) return;   // the rest takes no gradient
#pragma unroll
      for (int z = 0; z < 8; ++z)
        sum[z] += DROP ? kept(bits[q / 4] >> (4 * (q & 3)), z, x[q][z]) : x[q][z];
    }
  }
  if (cur >= j.rows || !mine) return;
  if (began_here && after != cur)
    put_row<TO>(a, j, cur, c, sum);
  else
    store8(part + (began_here ? a.dimp : 0), sum);
}

// A handful of tokens and a small table: one launch, whose workgroups each sort the tokens in LDS
// and then take SMALL_ROWS rows of a table, a wave a row, to clear or to add up.  256 tokens
// against the three launches, dim 768: 15.2 / 20.1 us for 2000 rows, 18.2 / 20.1 for 8000,
// 21.0 / 21.6 for 16000, 37.2 / 32.0 for 50257, where every workgroup's own sort is in the way of
// the clearing; dim 1280: 18.6 / 19.9 for 2000, 20.2 / 19.8 for 4000, 24.1 / 21.6 for 8000.
constexpr int SMALL_TOKENS = 256, SMALL_ROWS = 16, SMALL_AHEAD = 8;
// 16 tokens, dim 768: 14.6 / 17.4 for 8000, 14.7 / 17.1 for 16000, 19.9 / 18.7 for 32000.
constexpr long long SMALL_TABLE = 6 << 20, SMALL_TABLE_FEW = 16 << 20;   // elements

template <class TG, class TO, bool DROP>
__global__ __launch_bounds__(256) void embed_grad_small(GradArgs a) {
  __shared__ int raw[SMALL_TOKENS], keys[SMALL_TOKENS], order[SMALL_TOKENS];
  __shared__ int first[SMALL_ROWS + 1];
  const int groups = (a.job[0].rows + SMALL_ROWS - 1) / SMALL_ROWS;
  const int jn = (int)blockIdx.x >= groups;
  const GradJob& j = a.job[jn];
  const int v0 = ((int)blockIdx.x - jn * groups) * SMALL_ROWS, n = a.tokens, t = threadIdx.x;
  if (j.ids) {
    const int mine = t < n ? sort_key(j, load_index(j.ids, a.is64, t)) : 0;
    raw[t] = mine;
    __syncthreads();
    int at = 0;
    for (int i = 0; i < n; ++i) at += raw[i] < mine + (i < t);
    if (t < n) {
      keys[at] = mine;
      order[at] = t;
    }
    __syncthreads();
    if (t <= SMALL_ROWS) first[t] = first_at(keys, 0, n, v0 + t);
  } else if (t <= SMALL_ROWS) {
    first[t] = (v0 + t < a.seq ? v0 + t : a.seq) * (n ? a.batch : 0);
  }
  __syncthreads();
  const RngKey rk = DROP ? rng_key(a.rng) : RngKey{};
  const int lane = t & 63;
  for (int r = t >> 6; r < SMALL_ROWS; r += 4) {
    const int v = v0 + r;
    if (v >= j.rows) return;
    const int s0 = __builtin_amdgcn_readfirstlane(first[r]);
    const int s1 = __builtin_amdgcn_readfirstlane(first[r + 1]);
    if (s0 == s1 && j.accumulate) continue;
    for (int c = lane * 8; c < a.dim && lane < a.lanes; c += 8 * a.lanes) {
      if (c + 8 > a.dim) c = a.dim - 8;   // overlaps its neighbour's, as in embed_grad
      float sum[8] = {};
      for (int s = s0; s < s1; s += SMALL_AHEAD) {
        Raw8<TG> x[SMALL_AHEAD];
#pragma unroll
        for (int q = 0; q < SMALL_AHEAD; ++q) {
          const int e = s + q < s1 ? s + q : s1 - 1;
          const int i = j.ids ? order[e] : (e % a.batch) * a.seq + e / a.batch;
          x[q].load((const TG*)a.g + (long long)i * a.gstride + c);
        }
#pragma unroll
        for (int q = 0; q < SMALL_AHEAD; ++q) {
          if (s + q >= s1) break;
          uint32_t bits = ~0u;
          if (DROP) {
            const int e = s + q;
            const int i = j.ids ? order[e] : (e % a.batch) * a.seq + e / a.batch;
            const unsigned long long f = (unsigned long long)i * a.dim + c;
            bits = a.dim & 7 ? keep_bits_at<true>(a.rng, rk, f) : keep_bits_at<false>(a.rng, rk, f);
          }
#pragma unroll
          for (int z = 0; z < 8; ++z) sum[z] += DROP ? kept(bits, z, x[q][z]) : x[q][z];
        }
      }
      put_row<TO>(a, j, v, c, sum);
    }
  }
}

// Tables narrower than eight columns, which no piece of a row fits: the same chunks and parts, by
// eight lanes a chunk, one a column.  Right for any such table, and made for none to be fast; but
// a thread has no more than one chunk's tokens to walk through, however often an id occurs:
// 200000 tokens of four columns take 50 us if all have one id and 69 with 50257 of them, where a
// thread for each element of the table took 33000 and 56 (and stopped adding at 2^24 ones).
constexpr int NARROW_CHUNKS = 32;   // a workgroup

template <class TG, class TO, bool DROP>
__global__ __launch_bounds__(256) void embed_grad_narrow(GradArgs a) {
  const int sums = a.job[0].reduce_groups + a.job[1].reduce_groups;
  int b = blockIdx.x;
  if (b >= sums) {
    b -= sums;
    const int second = b >= a.job[0].fill_groups;
    clear_rows<TO>(a, a.job[second], second ? b - a.job[0].fill_groups : b);
    return;
  }
  const int jn = b >= a.job[0].reduce_groups;
  const GradJob& j = a.job[jn];
  if (jn) b -= a.job[0].reduce_groups;
  const int c = threadIdx.x & 7, chunk = b * NARROW_CHUNKS + (int)(threadIdx.x >> 3);
  if (chunk >= j.chunks || c >= a.dim) return;
  const int s0 = chunk * CHUNK, s1 = a.tokens - s0 < CHUNK ? a.tokens : s0 + CHUNK;
  const int before = s0 ? key_at(a, j, s0 - 1) : -1;
  const int after = s1 < a.tokens ? key_at(a, j, s1) : -1;
  const RngKey rk = DROP ? rng_key(a.rng) : RngKey{};
  float* part = j.part + (long long)chunk * 2 * a.dimp + c;
  auto put = [&](int row, float sum) {
    TO* o = (TO*)j.out + (long long)row * a.dim + c;
    *o = (TO)fmaf(sum, j.scale, j.accumulate ? (float)*o : 0.f);
  };
  float sum = 0.f;
  int cur = key_at(a, j, s0);
  bool began_here = cur != before;
  constexpr int AHEAD = 8;
  for (int e = s0; e < s1; e += AHEAD) {
    int key[AHEAD];
    long long tok[AHEAD];
    float x[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int s = e + q < s1 ? e + q : s1 - 1;
      key[q] = key_at(a, j, s);
      tok[q] = token_at(a, j, s);
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) x[q] = (float)((const TG*)a.g)[tok[q] * a.gstride + c];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (e + q >= s1) break;
      if (key[q] != cur) {
        if (began_here) put(cur, sum); else *part = sum;
        cur = key[q];
        began_here = true;
        sum = 0.f;
      }
      if (cur >= j.rows) return;   // the rest takes no gradient
      const unsigned long long f = (unsigned long long)(tok[q] * a.dim + c);
      sum += DROP ? kept(keep_bits(a.rng, rk, f >> 3), (int)(f & 7), x[q]) : x[q];
    }
  }
  if (cur >= j.rows) return;
  if (began_here && after != cur)
    put(cur, sum);
  else
    part[began_here ? a.dimp : 0] = sum;
}

// The ids that reach over a chunk's end: the part in the chunk where an id begins and those of
// the chunks that it fills or ends in, spread over four waves and added in their order.  5 us for
// 8192 tokens, 8.5 for 32768: the latency of a few dependent reads.
constexpr int JOIN_WAVES = 4;

template <class TO>
__global__ __launch_bounds__(64 * JOIN_WAVES) void embed_join(GradArgs a) {
  __shared__ float lds[JOIN_WAVES][64][9];
  const GradJob& j = a.job[blockIdx.z + !a.job[0].spans];
  const int chunk = blockIdx.x;
  const int end = (chunk + 1) * CHUNK, id = key_at(a, j, end - 1);
  if (id >= j.rows || key_at(a, j, end) != id) return;
  if (chunk && key_at(a, j, chunk * CHUNK - 1) == id) return;   // began before
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int c = (blockIdx.y * a.lanes + lane) * 8;
  const bool mine = lane < a.lanes && c < a.dim;
  c = mine && c + 8 <= a.dim ? c : a.dim - 8;
  // the id has a part in every chunk from here on whose first id it is; the sorted list says at
  // once of 64 chunks whether they are
  int last = chunk + 1;
  for (;;) {
    const int q = last + 1 + lane;
    const unsigned long long m =
        __ballot(q < j.chunks && key_at(a, j, (q < j.chunks ? q : chunk) * CHUNK) == id);
    last += m == ~0ull ? 64 : __builtin_ctzll(~m);
    if (m != ~0ull) break;
  }
  float sum[8] = {};
  const float* part = j.part + c;
#pragma unroll 4
  for (int q = chunk + 1 + wave; q <= last; q += JOIN_WAVES) {
    float x[8];
    load8(part + (long long)q * 2 * a.dimp, x);
#pragma unroll
    for (int z = 0; z < 8; ++z) sum[z] += x[z];
  }
#pragma unroll
  for (int z = 0; z < 8; ++z) lds[wave][lane][z] = sum[z];
  __syncthreads();
  if (wave || !mine) return;
  load8(j.part + ((long long)chunk * 2 + 1) * a.dimp + c, sum);
  for (int w = 0; w < JOIN_WAVES; ++w)
#pragma unroll
    for (int z = 0; z < 8; ++z) sum[z] += lds[w][lane][z];
  put_row<TO>(a, j, id, c, sum);
}

// ... of the narrow tables: 32 parts at a time, one column a lane
template <class TO>
__global__ __launch_bounds__(256) void embed_join_narrow(GradArgs a) {
  constexpr int PARTS = 256 / 8;
  __shared__ float lds[PARTS][8];
  const GradJob& j = a.job[blockIdx.z + !a.job[0].spans];
  const int chunk = blockIdx.x;
  const int end = (chunk + 1) * CHUNK, id = key_at(a, j, end - 1);
  if (id >= j.rows || key_at(a, j, end) != id) return;
  if (chunk && key_at(a, j, chunk * CHUNK - 1) == id) return;   // began before
  // the chunk with the id's last token
  const int last = ((j.ids ? first_at(j.keys, end, a.tokens, id + 1) : (id + 1) * a.batch) - 1) /
                   CHUNK;
  const int c = threadIdx.x & 7, p = threadIdx.x >> 3;
  const float* part = j.part + c;
  float sum = 0.f;
#pragma unroll 4
  for (int q = chunk + 1 + p; q <= last; q += PARTS) sum += part[(long long)q * 2 * a.dimp];
  lds[p][c] = sum;
  __syncthreads();
  if (p || c >= a.dim) return;
  sum = part[((long long)chunk * 2 + 1) * a.dimp];
  for (int q = 0; q < PARTS; ++q) sum += lds[q][c];
  TO* o = (TO*)j.out + (long long)id * a.dim + c;
  *o = (TO)fmaf(sum, j.scale, j.accumulate ? (float)*o : 0.f);
}

template <class TW, class TO, bool POS, bool DROP>
static void launch_rows(hipStream_t stream, const EmbedArgs& a) {
  const long long groups = (a.tokens + (256 >> a.log_lanes) - 1) / (256 >> a.log_lanes);
  const dim3 grid((unsigned)(groups < (1 << 22) ? groups : (1 << 22))), block(256);
  if (a.dim < 8)
    hipLaunchKernelGGL((embed_rows<TW, TO, POS, DROP, true, true>), grid, block, 0, stream, a);
  else if (a.dim & 7)
    hipLaunchKernelGGL((embed_rows<TW, TO, POS, DROP, true, false>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((embed_rows<TW, TO, POS, DROP, false, false>), grid, block, 0, stream, a);
}
template <class TW, class TO>
static void launch_rows(hipStream_t stream, const EmbedArgs& a) {
  if (a.p && a.rng.cut)
    launch_rows<TW, TO, true, true>(stream, a);
  else if (a.p)
    launch_rows<TW, TO, true, false>(stream, a);
  else if (a.rng.cut)
    launch_rows<TW, TO, false, true>(stream, a);
  else
    launch_rows<TW, TO, false, false>(stream, a);
}

template <class TG, class TO, bool DROP>
static void launch_grad(hipStream_t stream, const GradArgs& a) {
  if (a.small) {
    const int groups = ceil_div(a.job[0].rows, SMALL_ROWS) + ceil_div(a.job[1].rows, SMALL_ROWS);
    hipLaunchKernelGGL((embed_grad_small<TG, TO, DROP>), dim3(groups), dim3(256), 0, stream, a);
    return;
  }
  const int groups = a.job[0].reduce_groups + a.job[1].reduce_groups + a.job[0].fill_groups +
                     a.job[1].fill_groups;
  if (groups == 0) return;   // no tokens to add
  if (a.dim < 8)
    hipLaunchKernelGGL((embed_grad_narrow<TG, TO, DROP>), dim3(groups), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((embed_grad<TG, TO, DROP>), dim3(groups), dim3(256), 0, stream, a);
}
template <class TG, class TO>
static void launch_grad(hipStream_t stream, const GradArgs& a) {
  if (a.rng.cut)
    launch_grad<TG, TO, true>(stream, a);
  else
    launch_grad<TG, TO, false>(stream, a);
}

// Lanes of a wave that take columns: such that the last wave of a row has two at least where the
// last lane's columns overlap its neighbour's.
static int grad_lanes(int dim) {
  const int pieces = ceil_div(dim, 8);
  int lanes = 64;
  while (pieces > 1 && (dim & 7) && pieces % lanes == 1) --lanes;
  return lanes;
}

// what a table's gradient takes of the workspace: sorted ids and tokens, the radix sort's other
// buffers and counts, the parts of ids that reach over chunks
struct GradSpace {
  size_t keys, order, keys2, order2, hist, part, bytes;
};
static GradSpace grad_space(long long tokens, int dim, bool sorted) {
  GradSpace g{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  const long long chunks = ceil_div(tokens, CHUNK);
  if (sorted) {
    g.keys = take(4 * (size_t)tokens);
    g.order = take(4 * (size_t)tokens);
    if (tokens > RANK_MAX) {
      g.keys2 = take(4 * (size_t)tokens);
      g.order2 = take(4 * (size_t)tokens);
      g.hist = take(4 * 256 * RADIX_RUNS);
    }
  }
  g.part = take((size_t)chunks * 2 * ((dim + 7) / 8 * 8) * 4);
  g.bytes = at;
  return g;
}

// Whether the gradients take one launch (embed_grad_small), and no workspace.
static bool small_grad(long long tokens, long long rows, int dim) {
  return dim >= 8 && tokens <= SMALL_TOKENS &&
         rows * dim <= (tokens <= CHUNK ? SMALL_TABLE_FEW : SMALL_TABLE);
}

static bool grad_shape(long long tokens, long long rows, long long pos_rows, int dim) {
  // launches stay below 2^32 threads
  return tokens >= 0 && tokens < (1LL << 27) && rows >= 0 && rows < (1LL << 27) &&
         pos_rows >= 0 && pos_rows < (1LL << 27) && dim >= 0 && dim <= (1 << 23) &&
         (tokens / CHUNK + 1) * (dim / 256 + 1) < (1LL << 25);
}

// One job: its buffers, and how many workgroups it takes.
static void grad_job(GradJob& j, const GradArgs& a, const void* ids, void* out, long long rows,
                     long long padding, float scale, int accumulate, char* ws,
                     const GradSpace& sp) {
  j.ids = ids;
  j.out = out;
  j.keys = (int*)(ws + sp.keys);
  j.order = (int*)(ws + sp.order);
  j.keys2 = (int*)(ws + sp.keys2);
  j.order2 = (int*)(ws + sp.order2);
  j.hist = (int*)(ws + sp.hist);
  j.part = (float*)(ws + sp.part);
  j.padding = padding;
  j.rows = (int)rows;
  j.scale = scale;
  j.accumulate = accumulate;
  j.chunks = ceil_div(a.tokens, CHUNK);
  j.reduce_groups = a.dim < 8 ? ceil_div(j.chunks, NARROW_CHUNKS)
                              : ceil_div((long long)j.chunks * a.ctiles, 4);
  const bool all_named = !ids && a.tokens > 0 && a.seq >= rows;
  j.fill_groups = accumulate || all_named ? 0 : ceil_div(rows, FILL_ROWS);
  j.spans = j.chunks > 1 && (ids || CHUNK % a.batch != 0);
}

}  // namespace dmh

using namespace dmh;

extern "C" {

int dmh_embedding(hipStream_t stream, const void* ids, int ids_64, long long tokens, int seq,
                  const void* weight, int dtype, long long vocab, int dim, long long w_rstride,
                  const void* pos_weight, long long pos_rows, long long p_rstride,
                  const void* positions, float scale, int cut, unsigned long long seed,
                  unsigned long long offset, const void* rng_state, void* out, int out_dtype) {
  if (tokens < 0 || vocab < 0 || dim < 0 || w_rstride < 0 || pos_rows < 0 || p_rstride < 0 ||
      !float_code(dtype) || !float_code(out_dtype) || cut < 0 || cut > 65536 ||
      tokens > (1LL << 40) || vocab > (1LL << 40) || dim > (1 << 30) ||   // columns are ints
      (tokens > 0 && pos_weight && !positions && seq < 1)) {
    set_error("dmh_embedding: bad arguments (tokens=%lld seq=%d vocab=%lld dim=%d dtypes=%d,%d "
              "cut=%d)", tokens, seq, vocab, dim, dtype, out_dtype, cut);
    return DMH_EINVAL;
  }
  if (tokens == 0 || dim == 0) return DMH_OK;
  if (!ids || !out || (!weight && vocab)) {
    set_error("dmh_embedding: null tensor");
    return DMH_EINVAL;
  }
  EmbedArgs a;
  a.ids = ids;
  a.pos = positions;
  a.w = weight;
  a.p = pos_weight;
  a.out = out;
  a.tokens = tokens;
  a.vocab = vocab;
  a.wstride = w_rstride;
  a.prows = pos_rows;
  a.pstride = p_rstride;
  a.is64 = ids_64 != 0;
  a.seq = seq;
  a.dim = dim;
  // the most lanes of those that leave the fewest idle in a row's last round
  const int pieces = dim < 8 ? dim : ceil_div(dim, 8);
  int best = 1 << 30;
  for (int l = 6; l >= 0; --l) {
    const int rounds = ceil_div(pieces, 1 << l);
    if (rounds > 8 && l < 6) break;
    if (rounds << l < best) {
      best = rounds << l;
      a.log_lanes = l;
      a.lanes = 1 << l;
    }
  }
  a.scale = scale;
  a.rng = make_rng(seed, offset, rng_state, cut);
  DMH_FOR_TYPE(dtype, TW, DMH_FOR_TYPE(out_dtype, TO, (launch_rows<TW, TO>(stream, a))))
  DMH_CHECK_LAUNCH("embed_rows");
  return DMH_OK;
}

int dmh_embedding_grad_workspace_size(long long tokens, long long rows, long long pos_rows,
                                      int dim, int positions, size_t* bytes) {
  if (!bytes || !grad_shape(tokens, rows, pos_rows, dim)) {
    set_error("dmh_embedding_grad_workspace_size: bad arguments (tokens=%lld rows=%lld,%lld "
              "dim=%d)", tokens, rows, pos_rows, dim);
    return DMH_EINVAL;
  }
  *bytes = small_grad(tokens, rows + pos_rows, dim)
               ? 0
               : (rows ? grad_space(tokens, dim, true).bytes : 0) +
                     (pos_rows ? grad_space(tokens, dim, positions != 0).bytes : 0);
  return DMH_OK;
}

int dmh_embedding_grad(hipStream_t stream, const void* ids, const void* positions, int ids_64,
                       long long tokens, int seq, const void* grad, int dtype,
                       long long g_rstride, int dim, long long padding_idx, float scale, int cut,
                       unsigned long long seed, unsigned long long offset, const void* rng_state,
                       void* out, long long rows, int accumulate, void* pos_out,
                       long long pos_rows, int pos_accumulate, int out_dtype, void* ws,
                       size_t ws_bytes) {
  const bool pos = pos_out && pos_rows > 0, tok = out && rows > 0;
  if (!grad_shape(tokens, rows, pos_rows, dim) || g_rstride < 0 || !float_code(dtype) ||
      !float_code(out_dtype) || cut < 0 || cut > 65536 ||
      (pos && !positions && tokens > 0 && (seq < 1 || tokens % seq != 0))) {
    set_error("dmh_embedding_grad: bad arguments (tokens=%lld seq=%d rows=%lld,%lld dim=%d "
              "dtypes=%d,%d cut=%d)", tokens, seq, rows, pos_rows, dim, dtype, out_dtype, cut);
    return DMH_EINVAL;
  }
  if ((!tok && !pos) || dim == 0) return DMH_OK;
  if (tokens > 0 && (!grad || (tok && !ids))) {
    set_error("dmh_embedding_grad: null tensor");
    return DMH_EINVAL;
  }
  const GradSpace ts = tok ? grad_space(tokens, dim, true) : GradSpace{};
  const GradSpace ps = pos ? grad_space(tokens, dim, positions != nullptr) : GradSpace{};
  size_t need;
  dmh_embedding_grad_workspace_size(tokens, tok ? rows : 0, pos ? pos_rows : 0, dim,
                                    positions != nullptr, &need);
  if (need > 0 && (!ws || ws_bytes < need)) {
    set_error("dmh_embedding_grad: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return DMH_EWORKSPACE;
  }
  GradArgs a{};
  a.g = grad;
  a.gstride = g_rstride;
  a.is64 = ids_64 != 0;
  a.tokens = (int)tokens;
  a.seq = seq < 1 ? 1 : seq;
  a.batch = a.tokens / a.seq < 1 ? 1 : a.tokens / a.seq;
  a.dim = dim;
  a.dimp = (dim + 7) / 8 * 8;
  a.lanes = grad_lanes(dim);
  a.ctiles = ceil_div(dim, 8 * a.lanes);
  a.rng = make_rng(seed, offset, rng_state, cut);
  if (tok)
    grad_job(a.job[0], a, ids, out, rows, padding_idx, scale * a.rng.scale, accumulate != 0,
             (char*)ws, ts);
  if (pos)
    grad_job(a.job[1], a, positions, pos_out, pos_rows, -1, a.rng.scale, pos_accumulate != 0,
             (char*)ws + ts.bytes, ps);
  const int sorts = (a.job[0].ids != nullptr) + (a.job[1].ids != nullptr);
  a.small = small_grad(tokens, (tok ? rows : 0) + (pos ? pos_rows : 0), dim);
  if (tokens > 0 && sorts && !a.small) {
    if (tokens <= RANK_MAX) {
      hipLaunchKernelGGL(embed_rank, dim3(ceil_div(tokens, RANK_TOKENS), sorts),
                         dim3(RANK_THREADS), 0, stream, a);
      DMH_CHECK_LAUNCH("embed_rank");
    } else {
      const long long most = rows > pos_rows ? rows : pos_rows;   // the largest key
      int passes = 1;
      while (most >> (8 * passes)) ++passes;
      const int runs = tokens > (long long)RADIX_RUNS * RADIX_ROUND
                           ? RADIX_RUNS : ceil_div(tokens, RADIX_ROUND);
      const dim3 grid(runs, sorts), block(256);
      for (int p = 0; p < passes; ++p) {
        const int parity = (passes - p) & 1;
        hipLaunchKernelGGL(radix_count, grid, block, 0, stream, a, p, runs, parity);
        hipLaunchKernelGGL(radix_move, grid, block, 0, stream, a, p, runs, parity);
        DMH_CHECK_LAUNCH("radix sort");
      }
    }
  }
  DMH_FOR_TYPE(dtype, TG, DMH_FOR_TYPE(out_dtype, TO, (launch_grad<TG, TO>(stream, a))))
  DMH_CHECK_LAUNCH("embed_grad");
  if (!a.small && (a.job[0].spans || a.job[1].spans)) {
    const int chunks = ceil_div(tokens, CHUNK);
    const dim3 grid(chunks - 1, a.ctiles, a.job[0].spans + a.job[1].spans);
    if (dim < 8) {
      DMH_FOR_TYPE(out_dtype, TO, hipLaunchKernelGGL((embed_join_narrow<TO>), grid, dim3(256), 0,
                                                     stream, a))
    } else {
      DMH_FOR_TYPE(out_dtype, TO, hipLaunchKernelGGL((embed_join<TO>), grid,
                                                     dim3(64 * JOIN_WAVES), 0, stream, a))
    }
    DMH_CHECK_LAUNCH("embed_join");
  }
  return DMH_OK;
}

}  // extern "C"
