// swarm_gated.hip — gated linear recurrence (include/swarmseq.h: swarm_gated_scan_*, swarm_gated_step).
//
//   c_t = f_t p_t + (1 - f_t) z_t,  p_t = keep_{t-1} c_{t-1},  h_t = o_t c_t,  f, o = sigmoid of their gates.
// With a_t = f_t keep_{t-1} a step is c -> a c + b, and steps compose: (A, B) then (a, b) is (a A, a B + b). The
// gradient E_t of c_{t-1} runs the same kind of recurrence backwards:
//   D_t = o_t dh_t + E_{t+1},  E_t = a_t D_t,
//   d xf = D (p - z) f (1 - f),  d xz = D (1 - f),  d xo = dh c o (1 - o),  d c0 = E_0.
// Padding steps are the identity: a = 1, nothing added, zero outputs.
//
// Memory bound: three gates are read and h is written (forward), gates and dh are read and three gradients are
// written (backward), for some twenty operations an element.
//
// A workgroup owns kChannels channels (groups of four; a group never crosses a sequence, a workgroup may) and walks
// its part of the length in tiles of 64 steps forward, 32 backward. A thread holds one group over a segment of four
// (two) consecutive steps in registers, composes it, the segments are joined in LDS from the tile's incoming state,
// and the thread runs its steps once more from the true state. So a tile is read once, all its steps' loads are in
// flight together, and the only serial part is the LDS join. The backward pass reads one saved state per
// SWARM_GATED_TILE steps and forms the others again, forwards, beside its own backward join.
// Tile and group follow from the registers: 16 gates of three blocks fill what lets three waves a SIMD stay
// resident. With groups of eight, tiles of 128 steps, or the next tile fetched ahead the registers spill, and 32 or
// 128 channels a workgroup were slower as well (64 x 1024 x 2048).
// Steps that are padding in every sequence of a workgroup are written and not read.
//
// Up to kShort steps need no tiles. Sequences of fewer than four channels go channel by channel, 16 steps
// a thread, where the forward kernel spills 136 to 140 bytes (100000 x 64 x 1 bf16: 74 + 138 us,
// 0.7 TB/s). Few channels (one long sequence) do not fill the card: then the length is split
// into chunks as well, a first kernel composes each chunk, and the main kernel's workgroups start from the chunks
// before theirs: the gates are read twice.
//
// Measured (a 4 GiB copy reaches 4.8 TB/s of reads and writes together on this card):
//   64 sequences x 1024 steps x 2048 channels, bf16, ragged: forward 205 us, backward 365 us, 4.3 and 4.5 TB/s
//   1 x 32768 x 1024, bf16: chunks 38 + forward 59 us, chunks 49 + backward 106 us (36 + 53, 44 + 96 at best); the main
//   kernels 4.6 and 4.4 TB/s
//   256 x 4 x 4096, bf16: 11 + 24 us;  one step, 81920 x 64 (step_kernel): float32 20.5 us, 6.1 TB/s,
//   bf16 and float16 14.5 us, 5.8 TB/s
#include <type_traits>

#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kChannels = 64;                  // channels of a workgroup
constexpr int kTile = SWARM_GATED_TILE;        // steps of a tile of the backward pass, and between saved states
constexpr int kFwdTile = 64;                   // steps of a tile of the forward pass
static_assert(kFwdTile % kTile == 0, "the forward pass saves a state at segment starts");
constexpr int kQuarters = kThreads / kChannels;   // threads that join one channel's segments
// Workgroups that fill the card, two on each of 256 CUs: with fewer the length is split. (768 to 2048 of them: the
// same or slower at 1 x 32768 x 1024.)
constexpr int64_t kFill = 512;
constexpr int64_t kLeastTiles = 4;             // of a chunk: a launch more costs what walking fewer tiles saves

template <int VV, int TILE>
struct Shape {
    static constexpr int V = VV;                       // channels of a group
    static constexpr int kGroups = kChannels / V;      // groups of a workgroup
    static constexpr int kSegs = kThreads / kGroups;   // segments of a tile
    static constexpr int kSteps = TILE / kSegs;       // steps of a segment
    static constexpr int kPart = kSegs / kQuarters;    // segments that one joining thread composes
};

struct ScanArgs {
    int64_t n, steps, U;
    const void* gates;
    int64_t gn, gt;
    const float* keep;
    const int64_t* lengths;
    int64_t groups;        // groups of channels in each sequence
    int64_t blocks;        // workgroups that hold all groups
    int64_t chunk_tiles;   // tiles of a chunk
    int64_t chunks;
    float* agg;            // [chunks][2][n][U]: a chunk's A and B
};

// The workgroup's place. Workgroups go to the eight XCDs in turn; with neighbours on one XCD, neighbouring channels
// share its L2 and are fetched together (64 x 1024 x 2048, bf16, ragged: forward 217 -> 203 us, backward 380 -> 360).
// Where the length is split as well that gains nothing (4 x 4096 x 1024, f32: 44 against 47 us forward).
__device__ __forceinline__ int64_t place_of(const ScanArgs& p) {
    const unsigned per = gridDim.x / 8, b = blockIdx.x;
    return p.chunks == 1 && b < per * 8 ? (b % 8) * per + b / 8 : b;
}

// What a thread works on: V channels of one sequence, from u on. The last group of a sequence starts at U - V, so
// that no vector load crosses a row's end: it may share channels with the one before, and both write the same.
// Threads behind the last group read what the last group reads, and write nothing.
struct Lane {
    int64_t i, u, len;
    bool exists;
};

template <int V>
__device__ __forceinline__ Lane lane_of(const ScanArgs& p, int64_t group) {
    Lane l;
    l.exists = group < p.n * p.groups;
    if (!l.exists) group = p.n * p.groups - 1;
    l.i = group / p.groups;
    l.u = (group - l.i * p.groups) * V;
    if (l.u > p.U - V) l.u = p.U - V;
    l.len = p.lengths ? p.lengths[l.i] : p.steps;
    if (l.len > p.steps) l.len = p.steps;
    if (l.len < 0) l.len = 0;
    return l;
}

// what the state is multiplied by before step t
__device__ __forceinline__ float keep_of(const ScanArgs& p, int64_t i, int64_t t) {
    return p.keep && t > 0 ? p.keep[i * p.steps + t - 1] : 1.0f;
}

// A thread's steps of one tile: R of the gate blocks (block r at column off[r]), with DH the gradient of h, and
// keep before each step. Steps behind the end read the last one again (step 0 of an empty sequence): no load is
// conditional, so all of them are in flight together, and their values are selected away.
template <typename T, int V, int kSteps, int R, bool DH>
struct Rows {
    Pack<T, V> x[R][kSteps];
    Pack<T, V> d[DH ? kSteps : 1];
    float keep[kSteps];

    // ALL: no step from t0 on is padding.
    template <bool ALL>
    __device__ __forceinline__ void load(const ScanArgs& p, const Lane& l, const T* g, const int64_t (&off)[R],
                                         const T* dh, int64_t dt, int64_t t0) {
        const int64_t end = l.len > 0 ? l.len - 1 : 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t t = ALL || t0 + s < end ? t0 + s : end;
            const T* q = g + t * p.gt;
#pragma unroll
            for (int r = 0; r < R; ++r) x[r][s].load(q + off[r]);
            if (DH) d[s].load(dh + t * dt);
            keep[s] = p.keep ? p.keep[l.i * p.steps + (t > 0 ? t - 1 : 0)] : 1.0f;
            if (t == 0) keep[s] = 1.0f;
        }
    }
};

__device__ __forceinline__ void compose(float& A, float& B, float a, float b) {
    B = a * B + b;
    A = a * A;
}

// The step that every sequence of the workgroup reaches, and the one that none passes.
struct Span {
    int64_t whole, live;
};

template <typename R>
__device__ __forceinline__ Span span_of(const ScanArgs& p, int64_t len, R& red) {
    if (!p.lengths) return {p.steps, p.steps};
    int64_t(*ends)[2] = reinterpret_cast<int64_t(*)[2]>(&red);
    Span s{len, len};
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int64_t least = __shfl_xor(s.whole, o), most = __shfl_xor(s.live, o);
        s.whole = least < s.whole ? least : s.whole;
        s.live = most > s.live ? most : s.live;
    }
    if (threadIdx.x % 64 == 0) ends[threadIdx.x / 64][0] = s.whole, ends[threadIdx.x / 64][1] = s.live;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) {
        s.whole = ends[w][0] < s.whole ? ends[w][0] : s.whole;
        s.live = ends[w][1] > s.live ? ends[w][1] : s.live;
    }
    __syncthreads();
    return s;
}

// (A, B) of the chunks [from, to) in their order along the walk, by the joining threads of a channel, in every one
__device__ __forceinline__ void chunks_before(const ScanArgs& p, int64_t at, int64_t first, int64_t count, int64_t dir,
                                              int quarter, float (*red)[kChannels][2], int ch, float& A, float& B) {
    A = 1.0f;
    B = 0.0f;
    const int64_t size = p.n * p.U;
    const int64_t k0 = count * quarter / kQuarters, k1 = count * (quarter + 1) / kQuarters;
    for (int64_t k = k0; k < k1; ++k) {
        const float* a = p.agg + (first + dir * k) * 2 * size + at;
        compose(A, B, a[0], a[size]);
    }
    red[quarter][ch][0] = A;
    red[quarter][ch][1] = B;
    __syncthreads();
    A = red[0][ch][0];
    B = red[0][ch][1];
    for (int q = 1; q < kQuarters; ++q) compose(A, B, red[q][ch][0], red[q][ch][1]);
    __syncthreads();
}

// A chunk's composition. Forward: of c; backward (BWD): of E, from its last step to its first.
template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kThreads, V == 1 ? 2 : 3) void chunk_kernel(ScanArgs p, const T* dh, int64_t dn, int64_t dt) {
    using S = Shape<V, kFwdTile>;
    __shared__ float ab[2][S::kSegs][kChannels];
    __shared__ __align__(8) float red[kQuarters][kChannels][2];
    const int64_t part = blockIdx.x / p.blocks, block = blockIdx.x - part * p.blocks;
    const int64_t chunk = BWD ? part + 1 : part;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<V>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const bool has_dh = BWD && dh;
    const T* dhp = has_dh ? dh + l.i * dn + l.u : g;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    float cA = 1.0f, cB = 0.0f;
    const int64_t off[2] = {0, (BWD ? 2 : 1) * p.U};
    auto start = [&](int64_t k) {      // the thread's first step of the walk's tile k
        return (chunk * p.chunk_tiles + (BWD ? p.chunk_tiles - 1 - k : k)) * kFwdTile + seg * S::kSteps;
    };
    for (int64_t k = 0; k < p.chunk_tiles; ++k) {
        const int64_t t0 = start(k);
        Rows<T, V, S::kSteps, 2, BWD> now;
        now.template load<false>(p, l, g, off, dhp, dt, t0);
        float A[V], B[V];
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
        for (int q = 0; q < S::kSteps; ++q) {
            const int s = BWD ? S::kSteps - 1 - q : q;
            const bool on = t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float f, m;
                sigmoid_pair<T>(now.x[0][s].get(j), f, m);
                const float y = now.x[1][s].get(j), a = f * now.keep[s];
                const float b = BWD ? a * (sigmoid<T>(y) * (has_dh ? now.d[s].get(j) : 0.0f)) : m * y;
                compose(A[j], B[j], on ? a : 1.0f, on ? b : 0.0f);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            ab[0][BWD ? S::kSegs - 1 - seg : seg][lane * V + j] = A[j];
            ab[1][BWD ? S::kSegs - 1 - seg : seg][lane * V + j] = B[j];
        }
        __syncthreads();
        float qA = 1.0f, qB = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s)
            compose(qA, qB, ab[0][quarter * S::kPart + s][ch], ab[1][quarter * S::kPart + s][ch]);
        red[quarter][ch][0] = qA;
        red[quarter][ch][1] = qB;
        __syncthreads();
        for (int q = 0; q < kQuarters; ++q) compose(cA, cB, red[q][ch][0], red[q][ch][1]);
    }
    if (quarter == 0) {
        const Lane jl = lane_of<V>(p, block * S::kGroups + ch / V);
        float* out = p.agg + chunk * 2 * p.n * p.U + jl.i * p.U + jl.u + ch % V;
        if (jl.exists) {
            out[0] = cA;
            out[p.n * p.U] = cB;
        }
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads, V == 1 ? 2 : 3) void scan_fwd_kernel(ScanArgs p, const float* __restrict__ c0, T* __restrict__ h,
                                                               float* __restrict__ c_last,
                                                               float* __restrict__ states) {
    using S = Shape<V, kFwdTile>;
    __shared__ float ab[2][S::kSegs][kChannels];
    __shared__ __align__(8) float red[kQuarters][kChannels][2];
    const int64_t place = place_of(p), chunk = place / p.blocks, block = place - chunk * p.blocks;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<V>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    const Lane jl = lane_of<V>(p, block * S::kGroups + ch / V);
    const int64_t at = jl.i * p.U + jl.u + ch % V;
    const int64_t tiles = (p.steps + kFwdTile - 1) / kFwdTile;
    const int64_t saved = SWARM_GATED_TILES(p.steps);
    const int64_t first = chunk * p.chunk_tiles;
    const int64_t last = first + p.chunk_tiles < tiles ? first + p.chunk_tiles : tiles;
    const int64_t off[3] = {0, p.U, 2 * p.U};
    const Span span = span_of(p, l.len, red);
    float carry = c0 ? c0[at] : 0.0f;      // the channel's state before the tile, in every joining thread
    if (chunk > 0) {
        float A, B;
        chunks_before(p, at, 0, chunk, 1, quarter, red, ch, A, B);
        carry = A * carry + B;
    }
    auto run = [&](int64_t tile, auto all) {
        constexpr bool ALL = decltype(all)::value;      // no step of the tile is padding
        const int64_t t0 = tile * kFwdTile + seg * S::kSteps;
        Rows<T, V, S::kSteps, 3, false> rows;
        rows.template load<ALL>(p, l, g, off, g, 0, t0);
        float a[S::kSteps][V], b[S::kSteps][V], A[V], B[V];
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const bool on = ALL || t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float f, m;
                sigmoid_pair<T>(rows.x[0][s].get(j), f, m);
                a[s][j] = on ? f * rows.keep[s] : 1.0f;
                b[s][j] = on ? m * rows.x[1][s].get(j) : 0.0f;
                compose(A[j], B[j], a[s][j], b[s][j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            ab[0][seg][lane * V + j] = A[j];
            ab[1][seg][lane * V + j] = B[j];
        }
        __syncthreads();
        float pA[S::kPart], pB[S::kPart], qA = 1.0f, qB = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            pA[s] = ab[0][quarter * S::kPart + s][ch];
            pB[s] = ab[1][quarter * S::kPart + s][ch];
            compose(qA, qB, pA[s], pB[s]);
        }
        red[quarter][ch][0] = qA;
        red[quarter][ch][1] = qB;
        __syncthreads();
        float c = carry;
#pragma unroll
        for (int q = 0; q < kQuarters; ++q) {
            if (q == quarter) c = carry;
            carry = red[q][ch][0] * carry + red[q][ch][1];
        }
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            const int first_step = (quarter * S::kPart + s) * S::kSteps;
            if (states && first_step % kTile == 0 && jl.exists && tile * kFwdTile + first_step < p.steps)
                states[(jl.i * saved + tile * (kFwdTile / kTile) + first_step / kTile) * p.U + jl.u + ch % V] = c;
            ab[0][quarter * S::kPart + s][ch] = c;
            c = pA[s] * c + pB[s];
        }
        __syncthreads();
        float now[V];
#pragma unroll
        for (int j = 0; j < V; ++j) now[j] = ab[0][seg][lane * V + j];
        T* out = h + (l.i * p.steps + t0) * p.U + l.u;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            float v[V];
            const bool on = ALL || t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                now[j] = a[s][j] * now[j] + b[s][j];
                v[j] = on ? sigmoid<T>(rows.x[2][s].get(j)) * now[j] : 0.0f;
            }
            Pack<T, V> w;
            w.set(v);
            if (l.exists && (ALL || t0 + s < p.steps)) w.store(out + s * p.U);
        }
        __syncthreads();
    };
    // padding of all sequences: the state stands still, and nothing is read
    auto pass = [&](int64_t tile) {
        const int64_t t0 = tile * kFwdTile + seg * S::kSteps;
        T* out = h + (l.i * p.steps + t0) * p.U + l.u;
        Pack<T, V> none;
        none.clear();
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
            if (l.exists && t0 + s < p.steps) none.store(out + s * p.U);
        if (states && quarter == 0 && jl.exists)
            for (int k = 0; k < kFwdTile / kTile; ++k)
                if (tile * kFwdTile + k * kTile < p.steps)
                    states[(jl.i * saved + tile * (kFwdTile / kTile) + k) * p.U + jl.u + ch % V] = carry;
    };
    for (int64_t tile = first; tile < last; ++tile) {
        if ((tile + 1) * kFwdTile <= span.whole) run(tile, std::true_type{});
        else if (tile * kFwdTile < span.live) run(tile, std::false_type{});
        else pass(tile);
    }
    if (chunk == p.chunks - 1 && quarter == 0 && jl.exists) c_last[at] = carry;
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads, V == 1 ? 2 : 3) void scan_bwd_kernel(ScanArgs p, const float* __restrict__ states, const T* dh,
                                                               int64_t dn, int64_t dt,
                                                               const float* __restrict__ d_last, T* __restrict__ dg,
                                                               float* __restrict__ d_c0) {
    using S = Shape<V, kTile>;
    __shared__ float ab[3][S::kSegs][kChannels];     // A, B and the gradient's B; then the states before and behind
    __shared__ __align__(8) float red[kQuarters][kChannels][3];
    float (*before)[kChannels][2] = reinterpret_cast<float (*)[kChannels][2]>(&red[0][0][0]);
    const int64_t place = place_of(p), chunk = place / p.blocks, block = place - chunk * p.blocks;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<V>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const T* dhp = dh ? dh + l.i * dn + l.u : g;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    const Lane jl = lane_of<V>(p, block * S::kGroups + ch / V);
    const int64_t at = jl.i * p.U + jl.u + ch % V;
    const int64_t tiles = (p.steps + kTile - 1) / kTile;
    const int64_t chunk_tiles = p.chunk_tiles * (kFwdTile / kTile), first = chunk * chunk_tiles;
    const int64_t last = first + chunk_tiles < tiles ? first + chunk_tiles : tiles;
    const int64_t off[3] = {0, p.U, 2 * p.U};
    const Span span = span_of(p, l.len, red);
    float carry = d_last ? d_last[at] : 0.0f;     // E behind the tile
    if (chunk < p.chunks - 1) {
        float A, B;
        chunks_before(p, at, p.chunks - 1, p.chunks - 1 - chunk, -1, quarter, before, ch, A, B);
        carry = A * carry + B;
    }
    auto run = [&](int64_t tile, auto all) {
        constexpr bool ALL = decltype(all)::value;
        const int64_t t0 = tile * kTile + seg * S::kSteps;
        const float start = states[(jl.i * tiles + tile) * p.U + jl.u + ch % V];
        Rows<T, V, S::kSteps, 3, true> rows;
        rows.template load<ALL>(p, l, g, off, dhp, dt, t0);
        {
            float A[V], B[V], G[V];
#pragma unroll
            for (int j = 0; j < V; ++j) A[j] = 1.0f, B[j] = 0.0f, G[j] = 0.0f;
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s) {
                const bool on = ALL || t0 + s < l.len;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float f, m;
                    sigmoid_pair<T>(rows.x[0][s].get(j), f, m);
                    const float a = on ? f * rows.keep[s] : 1.0f;
                    const float od = sigmoid<T>(rows.x[2][s].get(j)) * (dh ? rows.d[s].get(j) : 0.0f);
                    B[j] = a * B[j] + (on ? m * rows.x[1][s].get(j) : 0.0f);
                    A[j] *= a;
                    // E at the segment's first step is the sum of a_0 .. a_s (o dh)_s
                    G[j] += on ? A[j] * od : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ab[0][seg][lane * V + j] = A[j];
                ab[1][seg][lane * V + j] = B[j];
                ab[2][seg][lane * V + j] = G[j];
            }
        }
        __syncthreads();
        float pA[S::kPart], pB[S::kPart], pG[S::kPart], qA = 1.0f, qB = 0.0f, qG = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            pA[s] = ab[0][quarter * S::kPart + s][ch];
            pB[s] = ab[1][quarter * S::kPart + s][ch];
            pG[s] = ab[2][quarter * S::kPart + s][ch];
            qB = pA[s] * qB + pB[s];
            qG += qA * pG[s];
            qA *= pA[s];
        }
        red[quarter][ch][0] = qA;
        red[quarter][ch][1] = qB;
        red[quarter][ch][2] = qG;
        __syncthreads();
        float c = start, E = carry;
#pragma unroll
        for (int q = 0; q < kQuarters; ++q)
            if (q < quarter) c = red[q][ch][0] * c + red[q][ch][1];
#pragma unroll
        for (int q = kQuarters - 1; q >= 0; --q) {
            if (q == quarter) E = carry;
            carry = red[q][ch][0] * carry + red[q][ch][2];
        }
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            ab[0][quarter * S::kPart + s][ch] = c;
            c = pA[s] * c + pB[s];
        }
#pragma unroll
        for (int s = S::kPart - 1; s >= 0; --s) {
            ab[1][quarter * S::kPart + s][ch] = E;
            E = pA[s] * E + pG[s];
        }
        __syncthreads();
        float now[V], back[V], cs[S::kSteps][V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            now[j] = ab[0][seg][lane * V + j];
            back[j] = ab[1][seg][lane * V + j];
        }
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const bool on = ALL || t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float f, m;
                sigmoid_pair<T>(rows.x[0][s].get(j), f, m);
                cs[s][j] = now[j] * rows.keep[s];
                now[j] = on ? f * cs[s][j] + m * rows.x[1][s].get(j) : now[j];
            }
        }
        T* out = dg + (l.i * p.steps + t0) * 3 * p.U + l.u;
#pragma unroll
        for (int s = S::kSteps - 1; s >= 0; --s) {
            const bool on = ALL || t0 + s < l.len;
            float vf[V], vz[V], vo[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float f, m, o, om;
                sigmoid_pair<T>(rows.x[0][s].get(j), f, m);
                sigmoid_pair<T>(rows.x[2][s].get(j), o, om);
                const float z = rows.x[1][s].get(j), pr = cs[s][j];
                const float cc = f * pr + m * z;
                const float od = o * (dh ? rows.d[s].get(j) : 0.0f);
                const float D = od + back[j];
                vf[j] = on ? D * (pr - z) * (f * m) : 0.0f;
                vz[j] = on ? D * m : 0.0f;
                vo[j] = on ? od * om * cc : 0.0f;
                back[j] = on ? f * rows.keep[s] * D : back[j];
            }
            T* w = out + s * 3 * p.U;
            Pack<T, V> wf, wz, wo;
            wf.set(vf), wz.set(vz), wo.set(vo);
            if (l.exists && (ALL || t0 + s < p.steps)) {
                wf.store(w);
                wz.store(w + p.U);
                wo.store(w + 2 * p.U);
            }
        }
        __syncthreads();
    };
    auto pass = [&](int64_t tile) {
        const int64_t t0 = tile * kTile + seg * S::kSteps;
        T* out = dg + (l.i * p.steps + t0) * 3 * p.U + l.u;
        Pack<T, V> none;
        none.clear();
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
            for (int r = 0; r < 3; ++r)
                if (l.exists && t0 + s < p.steps) none.store(out + (s * 3 + r) * p.U);
    };
    for (int64_t tile = last - 1; tile >= first; --tile) {
        if ((tile + 1) * kTile <= span.whole) run(tile, std::true_type{});
        else if (tile * kTile < span.live) run(tile, std::false_type{});
        else pass(tile);
    }
    if (d_c0 && chunk == 0 && quarter == 0 && jl.exists) d_c0[at] = carry;
}

// Sequences of at most kShort steps: a thread walks its channels through all of them, with every step's loads in
// flight at once and nothing to join. 16 steps fill its registers, and beat the tile kernels, most of whose threads
// then have no step (us, forward + backward, against tiles): 256 x 16 x 4032 bf16 39 + 68 / 90 + 95, 256 x 12 x 4064 bf16
// 25 + 57 / 90 + 96, 256 x 16 x 2000 float32 37 + 47 / 53 + 56. From 17 steps on the tiles' time is what it takes: 91 + 96 for
// 256 x 17 x 4000 bf16.
constexpr int kShort = 16;

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void short_fwd_kernel(ScanArgs p, const float* __restrict__ c0, T* __restrict__ h,
                                                             float* __restrict__ c_last, float* __restrict__ states) {
    const Lane l = lane_of<V>(p, (int64_t)blockIdx.x * kThreads + threadIdx.x);
    if (!l.exists) return;
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const int64_t at = l.i * p.U + l.u;
    Pack<T, V> xf[kShort], xz[kShort], xo[kShort];
    float keep[kShort], c[V];
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.steps) continue;
        const int64_t k = t < l.len ? t : (l.len > 0 ? l.len - 1 : 0);
        const T* q = g + k * p.gt;
        xf[t].load(q);
        xz[t].load(q + p.U);
        xo[t].load(q + 2 * p.U);
        keep[t] = keep_of(p, l.i, k);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = c0 ? c0[at + j] : 0.0f;
    if (states)
#pragma unroll
        for (int j = 0; j < V; ++j) states[at + j] = c[j];
    T* out = h + l.i * p.steps * p.U + l.u;
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.steps) continue;
        const bool on = t < l.len;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float f, m;
            sigmoid_pair<T>(xf[t].get(j), f, m);
            const float now = f * (c[j] * keep[t]) + m * xz[t].get(j);
            c[j] = on ? now : c[j];
            v[j] = on ? sigmoid<T>(xo[t].get(j)) * now : 0.0f;
        }
        Pack<T, V> w;
        w.set(v);
        w.store(out + t * p.U);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) c_last[at + j] = c[j];
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void short_bwd_kernel(ScanArgs p, const float* __restrict__ states, const T* dh,
                                                             int64_t dn, int64_t dt,
                                                             const float* __restrict__ d_last, T* __restrict__ dg,
                                                             float* __restrict__ d_c0) {
    const Lane l = lane_of<V>(p, (int64_t)blockIdx.x * kThreads + threadIdx.x);
    if (!l.exists) return;
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const T* dhp = dh ? dh + l.i * dn + l.u : g;
    const int64_t at = l.i * p.U + l.u;
    Pack<T, V> xf[kShort], xz[kShort], xo[kShort], d[kShort];
    float keep[kShort], pr[kShort][V], c[V], E[V];
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.steps) continue;
        const int64_t k = t < l.len ? t : (l.len > 0 ? l.len - 1 : 0);
        const T* q = g + k * p.gt;
        xf[t].load(q);
        xz[t].load(q + p.U);
        xo[t].load(q + 2 * p.U);
        d[t].load(dhp + k * dt);
        keep[t] = keep_of(p, l.i, k);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c[j] = states[at + j];
        E[j] = d_last ? d_last[at + j] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.steps) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float f, m;
            sigmoid_pair<T>(xf[t].get(j), f, m);
            pr[t][j] = c[j] * keep[t];
            c[j] = t < l.len ? f * pr[t][j] + m * xz[t].get(j) : c[j];
        }
    }
    T* out = dg + l.i * p.steps * 3 * p.U + l.u;
#pragma unroll
    for (int t = kShort - 1; t >= 0; --t) {
        if (t >= p.steps) continue;
        const bool on = t < l.len;
        float vf[V], vz[V], vo[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float f, m, o, om;
            sigmoid_pair<T>(xf[t].get(j), f, m);
            sigmoid_pair<T>(xo[t].get(j), o, om);
            const float z = xz[t].get(j), od = o * (dh ? d[t].get(j) : 0.0f), D = od + E[j];
            vf[j] = on ? D * (pr[t][j] - z) * (f * m) : 0.0f;
            vz[j] = on ? D * m : 0.0f;
            vo[j] = on ? od * om * (f * pr[t][j] + m * z) : 0.0f;
            E[j] = on ? f * keep[t] * D : E[j];
        }
        Pack<T, V> wf, wz, wo;
        wf.set(vf), wz.set(vz), wo.set(vo);
        T* w = out + t * 3 * p.U;
        wf.store(w);
        wz.store(w + p.U);
        wo.store(w + 2 * p.U);
    }
    if (d_c0)
#pragma unroll
        for (int j = 0; j < V; ++j) d_c0[at + j] = E[j];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void step_kernel(int64_t rows, int64_t U, const T* __restrict__ gates, int64_t gr,
                                                        const float* c, const float* __restrict__ keep,
                                                        T* __restrict__ h, float* c_out) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (id >= rows * U) return;
    const int64_t i = id / U, u = id - i * U;
    const T* g = gates + i * gr + u;
    float f, b;
    sigmoid_pair<T>((float)g[0], f, b);
    const float p = keep ? c[id] * keep[i] : c[id];
    const float now = f * p + b * (float)g[U];
    c_out[id] = now;
    h[id] = (T)(sigmoid<T>((float)g[2 * U]) * now);
}

// Vectors of kWide channels; sequences narrower than that go channel by channel.
constexpr int kWide = 4;
int64_t width_of(int64_t U) { return U >= kWide ? kWide : 1; }

// How the length is split: whole tiles, as many chunks as fill the card together with the channels.
void split(ScanArgs& p) {
    const int64_t V = width_of(p.U), per_block = kChannels / V;
    p.groups = (p.U + V - 1) / V;
    p.blocks = (p.n * p.groups + per_block - 1) / per_block;
    const int64_t tiles = (p.steps + kFwdTile - 1) / kFwdTile;
    int64_t want = p.blocks >= kFill ? 1 : (kFill + p.blocks - 1) / p.blocks;
    if (want > tiles / kLeastTiles) want = tiles / kLeastTiles > 0 ? tiles / kLeastTiles : 1;
    p.chunk_tiles = (tiles + want - 1) / want;
    p.chunks = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
}

// Short sequences: 8 bytes of channels a thread, so that their steps fit its registers.
template <typename F>
void with_short(int32_t dtype, int64_t U, F&& fn) {
    with_type(dtype, [&](auto e) {
        constexpr int V = 8 / sizeof(e);
        if (U >= V) fn(e, std::integral_constant<int, V>{});
        else fn(e, std::integral_constant<int, 1>{});
    });
}

// Groups of V channels in each sequence, and the workgroups with a thread for each.
void short_grid(ScanArgs& p, int64_t V) {
    p.groups = (p.U + V - 1) / V;
    p.blocks = (p.n * p.groups + kThreads - 1) / kThreads;
}

// Sequences of a launch: all, unless their threads (four for each channel, at most) pass what a grid counts, and
// then equal parts, each of which fills the card without its length split. 0: not even one.
int64_t part_of(int64_t n, int64_t U) {
    const int64_t most = (kLaunch - kThreads) / (kThreads / kChannels) / ((U + kWide - 1) / kWide * kWide);
    if (most < 1) return 0;
    const int64_t parts = (n + most - 1) / most;
    return (n + parts - 1) / parts;
}

// p, moved on by elements of a type
void* ahead(const void* p, int64_t elements, int32_t dtype) {
    return p ? const_cast<char*>(static_cast<const char*>(p)) + elements * (dtype == SWARM_F32 ? 4 : 2) : nullptr;
}
template <typename T>
T* ahead(T* p, int64_t elements) {
    return p ? p + elements : nullptr;
}

template <typename F>
void with_type_and_width(int32_t dtype, int64_t U, F&& fn) {
    with_type(dtype, [&](auto e) {
        if (width_of(U) == kWide) fn(e, std::integral_constant<int, kWide>{});
        else fn(e, std::integral_constant<int, 1>{});
    });
}

// One launch's sequences.
int32_t forward_part(int32_t dtype, const ScanArgs& args, const float* c0, void* h, float* c_last, float* tile_states,
                     hipStream_t st) {
    ScanArgs p = args;
    if (p.steps <= kShort) {
        with_short(dtype, p.U, [&](auto e, auto v) {
            using E = decltype(e);
            constexpr int V = decltype(v)::value;
            short_grid(p, V);
            short_fwd_kernel<E, V><<<(unsigned)p.blocks, kThreads, 0, st>>>(p, c0, static_cast<E*>(h), c_last,
                                                                          tile_states);
        });
        return swarm::record_hip_status();
    }
    split(p);
    if (p.chunks > 1 && !p.agg) return SWARM_ERR_ARG;
    with_type_and_width(dtype, p.U, [&](auto e, auto v) {
        using E = decltype(e);
        constexpr int V = decltype(v)::value;
        if (p.chunks > 1)
            chunk_kernel<E, V, false><<<(unsigned)(p.blocks * (p.chunks - 1)), kThreads, 0, st>>>(p, nullptr, 0, 0);
        scan_fwd_kernel<E, V><<<(unsigned)(p.blocks * p.chunks), kThreads, 0, st>>>(p, c0, static_cast<E*>(h), c_last,
                                                                                  tile_states);
    });
    return swarm::record_hip_status();
}

int32_t backward_part(int32_t dtype, const ScanArgs& args, const float* tile_states, const void* d_h, int64_t d_h_n,
                      int64_t d_h_t, const float* d_last, void* d_gates, float* d_c0, hipStream_t st) {
    ScanArgs p = args;
    const int64_t dt = d_h ? d_h_t : p.gt;      // without d_h the loads go to the gates
    if (p.steps <= kShort) {
        with_short(dtype, p.U, [&](auto e, auto v) {
            using E = decltype(e);
            constexpr int V = decltype(v)::value;
            short_grid(p, V);
            short_bwd_kernel<E, V><<<(unsigned)p.blocks, kThreads, 0, st>>>(
                p, tile_states, static_cast<const E*>(d_h), d_h_n, dt, d_last, static_cast<E*>(d_gates), d_c0);
        });
        return swarm::record_hip_status();
    }
    split(p);
    if (p.chunks > 1 && !p.agg) return SWARM_ERR_ARG;
    with_type_and_width(dtype, p.U, [&](auto e, auto v) {
        using E = decltype(e);
        constexpr int V = decltype(v)::value;
        const E* dh = static_cast<const E*>(d_h);
        if (p.chunks > 1)
            chunk_kernel<E, V, true><<<(unsigned)(p.blocks * (p.chunks - 1)), kThreads, 0, st>>>(p, dh, d_h_n, dt);
        scan_bwd_kernel<E, V><<<(unsigned)(p.blocks * p.chunks), kThreads, 0, st>>>(p, tile_states, dh, d_h_n, dt, d_last,
                                                                                  static_cast<E*>(d_gates), d_c0);
    });
    return swarm::record_hip_status();
}

}  // namespace

extern "C" {

int64_t swarm_gated_scan_workspace(int64_t n, int64_t T, int64_t U) {
    if (n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return 0;
    ScanArgs p{n, T, U};
    split(p);
    return p.chunks > 1 ? p.chunks * 2 * n * U : 0;
}

int32_t swarm_gated_scan_forward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                 int64_t gates_t, const float* c0, const float* keep, const int64_t* lengths, void* h,
                                 float* c_last, float* tile_states, float* work, void* stream) {
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    const int64_t part = part_of(n, U);
    if (!gates || !h || !c_last || gates_t < 0 || gates_n < 0 || part < 1) return SWARM_ERR_ARG;
    for (int64_t i = 0; i < n; i += part) {
        const ScanArgs p{n - i < part ? n - i : part, T, U, ahead(gates, i * gates_n, dtype), gates_n, gates_t,
                         ahead(keep, i * T), ahead(lengths, i), 0, 0, 0, 0, work};
        const int32_t rc = forward_part(dtype, p, ahead(c0, i * U), ahead(h, i * T * U, dtype), c_last + i * U,
                                        ahead(tile_states, i * SWARM_GATED_TILES(T) * U),
                                        static_cast<hipStream_t>(stream));
        if (rc != SWARM_OK) return rc;
    }
    return SWARM_OK;
}

int32_t swarm_gated_scan_backward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                  int64_t gates_t, const float* keep, const int64_t* lengths,
                                  const float* tile_states, const void* d_h, int64_t d_h_n, int64_t d_h_t,
                                  const float* d_last, void* d_gates, float* d_c0, float* work, void* stream) {
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    const int64_t part = part_of(n, U);
    if (!gates || !tile_states || !d_gates || gates_t < 0 || gates_n < 0 || d_h_n < 0 || d_h_t < 0 || part < 1)
        return SWARM_ERR_ARG;
    for (int64_t i = 0; i < n; i += part) {
        const ScanArgs p{n - i < part ? n - i : part, T, U, ahead(gates, i * gates_n, dtype), gates_n, gates_t,
                         ahead(keep, i * T), ahead(lengths, i), 0, 0, 0, 0, work};
        const int32_t rc = backward_part(dtype, p, tile_states + i * SWARM_GATED_TILES(T) * U,
                                         ahead(d_h, i * d_h_n, dtype), d_h_n, d_h_t, ahead(d_last, i * U),
                                         ahead(d_gates, i * T * 3 * U, dtype), ahead(d_c0, i * U),
                                         static_cast<hipStream_t>(stream));
        if (rc != SWARM_OK) return rc;
    }
    return SWARM_OK;
}

int32_t swarm_gated_step(int32_t dtype, int64_t rows, int64_t U, const void* gates, int64_t gates_row, const float* c,
                         const float* keep, void* h, float* c_out, void* stream) {
    if (!known_type(dtype) || rows < 0 || U < 1 || !sane(rows, U)) return SWARM_ERR_ARG;
    if (rows == 0) return SWARM_OK;
    const int64_t most = (kLaunch - kThreads) / U;      // rows of a launch
    if (!gates || !c || !h || !c_out || gates_row < 0 || most < 1) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        for (int64_t r = 0; r < rows; r += most) {
            const int64_t part = rows - r < most ? rows - r : most;
            step_kernel<E><<<(unsigned)((part * U + kThreads - 1) / kThreads), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                part, U, static_cast<const E*>(gates) + r * gates_row, gates_row, c + r * U, ahead(keep, r),
                static_cast<E*>(h) + r * U, c_out + r * U);
        }
    });
    return swarm::record_hip_status();
}

}  // extern "C"
