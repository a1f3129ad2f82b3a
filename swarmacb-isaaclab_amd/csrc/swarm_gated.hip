// swarm_gated.hip — gated linear recurrence (include/swarmseq.h: swarm_gated_scan_*, swarm_gated_step).
//
//   c_t = f_t p_t + (1 - f_t) z_t,  p_t = keep_{t-1} c_{t-1},  h_t = o_t c_t,  f, o = sigmoid of their gates.
// With a_t = f_t keep_{t-1} a step is c -> a c + b, and steps compose: (A, B) then (a, b) is (a A, a B + b). The
// gradient E_t of c_{t-1} runs the same kind of recurrence backwards:
//   D_t = o_t dh_t + E_{t+1},  E_t = a_t D_t,
//   d xf = D (p - z) f (1 - f),  d xz = D (1 - f),  d xo = dh c o (1 - o),  d c0 = E_0.
// Padding steps are the identity: a = 1, nothing added, zero outputs.
//
// A workgroup owns kChannels channels (16-byte groups of them; a group never crosses a sequence, a workgroup may)
// and walks its part of the length in tiles of SWARM_GATED_TILE steps. A thread holds one group over a segment of
// a few consecutive steps in registers, composes it, the segments are joined in LDS from the tile's incoming
// state, and the thread runs its steps once more from the true state. So a tile is read once, all its steps'
// loads are in flight together, and the only serial part is the LDS join. The backward pass reads one saved state
// per tile and forms the others again, forwards, beside its own backward join.
//
// Few channels (one long sequence) do not fill the card: then the length is split into chunks as well, a first
// kernel composes each chunk, and the main kernel's workgroups start from the chunks before theirs.
#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kChannels = 64;                  // channels of a workgroup
constexpr int kTile = SWARM_GATED_TILE;        // steps of a tile
constexpr int kQuarters = kThreads / kChannels;   // threads that join one channel's segments
constexpr int64_t kFill = 1024;                // workgroups that fill the card (four on each of 256 CUs)

template <typename T>
struct Shape {
    static constexpr int V = Pack<T>::V;               // channels of a group
    static constexpr int kGroups = kChannels / V;      // groups of a workgroup
    static constexpr int kSegs = kThreads / kGroups;   // segments of a tile
    static constexpr int kSteps = kTile / kSegs;       // steps of a segment
    static constexpr int kPart = kSegs / kQuarters;    // segments that one joining thread composes
};

struct ScanArgs {
    int64_t n, steps, U;
    const void* gates;
    int64_t gn, gt;
    const float* keep;
    const int64_t* lengths;
    int64_t groups;        // groups of channels in each sequence
    int64_t chunk_tiles;   // tiles of a chunk
    int64_t chunks;
    float* agg;            // [chunks][2][n][U]: a chunk's A and B
};

// What a thread works on: a group of channels of one sequence.
struct Lane {
    int64_t i, u, len;
    int valid;             // channels of the group that exist
};

template <typename T>
__device__ __forceinline__ Lane lane_of(const ScanArgs& p, int64_t group) {
    Lane l;
    l.i = group / p.groups;
    l.u = (group - l.i * p.groups) * Pack<T>::V;
    l.valid = 0;
    l.len = 0;
    if (l.i < p.n) {
        l.valid = p.U - l.u < Pack<T>::V ? (int)(p.U - l.u) : Pack<T>::V;
        l.len = p.lengths ? p.lengths[l.i] : p.steps;
        if (l.len > p.steps) l.len = p.steps;
    }
    return l;
}

// keep before step t
__device__ __forceinline__ float keep_of(const ScanArgs& p, int64_t i, int64_t t) {
    return p.keep && t > 0 ? p.keep[i * p.steps + t - 1] : 1.0f;
}

__device__ __forceinline__ void compose(float& A, float& B, float a, float b) {
    B = a * B + b;
    A = a * A;
}

// (A, B) of the chunks [from, to) in their order along the walk, by the joining threads of a channel, in every one
__device__ __forceinline__ void chunks_before(const ScanArgs& p, int64_t at, int64_t first, int64_t count, int64_t dir,
                                              int quarter, float (*red)[kChannels][2], int ch, bool exists, float& A,
                                              float& B) {
    A = 1.0f;
    B = 0.0f;
    const int64_t size = p.n * p.U;
    const int64_t k0 = count * quarter / kQuarters, k1 = count * (quarter + 1) / kQuarters;
    if (exists)
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
template <typename T, bool BWD>
__global__ __launch_bounds__(kThreads) void chunk_kernel(ScanArgs p, const T* __restrict__ dh, int64_t dn, int64_t dt) {
    using S = Shape<T>;
    __shared__ float ab[S::kSegs][kChannels][2];
    __shared__ float red[kQuarters][kChannels][2];
    const int64_t blocks = (p.n * p.groups + S::kGroups - 1) / S::kGroups;
    const int64_t part = blockIdx.x / blocks, block = blockIdx.x - part * blocks;
    const int64_t chunk = BWD ? part + 1 : part;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<T>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    const Lane jl = lane_of<T>(p, block * S::kGroups + ch / S::V);
    const bool exists = ch % S::V < jl.valid;
    float cA = 1.0f, cB = 0.0f;
    for (int64_t k = 0; k < p.chunk_tiles; ++k) {
        const int64_t tile = chunk * p.chunk_tiles + (BWD ? p.chunk_tiles - 1 - k : k);
        const int64_t t0 = tile * kTile + seg * S::kSteps;
        Pack<T> x[S::kSteps], y[S::kSteps], d[BWD ? S::kSteps : 1];
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const int valid = t0 + s < l.len ? l.valid : 0;
            x[s] = load_pack(g + (t0 + s) * p.gt, valid);
            y[s] = load_pack(g + (t0 + s) * p.gt + (BWD ? 2 : 1) * p.U, valid);
            if (BWD) d[s] = load_pack(dh + l.i * dn + (t0 + s) * dt + l.u, dh ? valid : 0);
        }
        float A[S::V], B[S::V];
#pragma unroll
        for (int j = 0; j < S::V; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
        for (int q = 0; q < S::kSteps; ++q) {
            const int s = BWD ? S::kSteps - 1 - q : q;
            if (t0 + s >= l.len) continue;
            const float kp = keep_of(p, l.i, t0 + s);
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                float f, b;
                sigmoid_pair((float)x[s].e[j], f, b);
                const float a = f * kp;
                compose(A[j], B[j], a, BWD ? a * (sigmoid((float)y[s].e[j]) * (float)d[s].e[j]) : b * (float)y[s].e[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
            ab[BWD ? S::kSegs - 1 - seg : seg][lane * S::V + j][0] = A[j];
            ab[BWD ? S::kSegs - 1 - seg : seg][lane * S::V + j][1] = B[j];
        }
        __syncthreads();
        float qA = 1.0f, qB = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            const float* e = ab[quarter * S::kPart + s][ch];
            compose(qA, qB, e[0], e[1]);
        }
        red[quarter][ch][0] = qA;
        red[quarter][ch][1] = qB;
        __syncthreads();
        for (int q = 0; q < kQuarters; ++q) compose(cA, cB, red[q][ch][0], red[q][ch][1]);
    }
    if (quarter == 0 && exists) {
        float* out = p.agg + chunk * 2 * p.n * p.U + jl.i * p.U + jl.u + ch % S::V;
        out[0] = cA;
        out[p.n * p.U] = cB;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void scan_fwd_kernel(ScanArgs p, const float* __restrict__ c0, T* __restrict__ h,
                                                            float* __restrict__ c_last, float* __restrict__ states) {
    using S = Shape<T>;
    __shared__ float ab[S::kSegs][kChannels][2];
    __shared__ float red[kQuarters][kChannels][2];
    const int64_t blocks = (p.n * p.groups + S::kGroups - 1) / S::kGroups;
    const int64_t chunk = blockIdx.x / blocks, block = blockIdx.x - chunk * blocks;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<T>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    const Lane jl = lane_of<T>(p, block * S::kGroups + ch / S::V);
    const bool exists = ch % S::V < jl.valid;
    const int64_t at = jl.i * p.U + jl.u + ch % S::V;
    const int64_t tiles = (p.steps + kTile - 1) / kTile;
    float carry = exists && c0 ? c0[at] : 0.0f;      // the channel's state before the tile, in every joining thread
    if (chunk > 0) {
        float A, B;
        chunks_before(p, at, 0, chunk, 1, quarter, red, ch, exists, A, B);
        carry = A * carry + B;
    }
    const int64_t first = chunk * p.chunk_tiles;
    const int64_t last = first + p.chunk_tiles < tiles ? first + p.chunk_tiles : tiles;
    for (int64_t tile = first; tile < last; ++tile) {
        const int64_t t0 = tile * kTile + seg * S::kSteps;
        Pack<T> xf[S::kSteps], xz[S::kSteps], xo[S::kSteps];
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const int valid = t0 + s < l.len ? l.valid : 0;
            const T* q = g + (t0 + s) * p.gt;
            xf[s] = load_pack(q, valid);
            xz[s] = load_pack(q + p.U, valid);
            xo[s] = load_pack(q + 2 * p.U, valid);
        }
        float a[S::kSteps][S::V], b[S::kSteps][S::V], A[S::V], B[S::V];
#pragma unroll
        for (int j = 0; j < S::V; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const bool on = t0 + s < l.len;
            const float kp = on ? keep_of(p, l.i, t0 + s) : 1.0f;
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                float f, m;
                sigmoid_pair((float)xf[s].e[j], f, m);
                a[s][j] = on ? f * kp : 1.0f;
                b[s][j] = on ? m * (float)xz[s].e[j] : 0.0f;
                compose(A[j], B[j], a[s][j], b[s][j]);
            }
        }
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
            ab[seg][lane * S::V + j][0] = A[j];
            ab[seg][lane * S::V + j][1] = B[j];
        }
        __syncthreads();
        float pA[S::kPart], pB[S::kPart], qA = 1.0f, qB = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            pA[s] = ab[quarter * S::kPart + s][ch][0];
            pB[s] = ab[quarter * S::kPart + s][ch][1];
            compose(qA, qB, pA[s], pB[s]);
        }
        red[quarter][ch][0] = qA;
        red[quarter][ch][1] = qB;
        __syncthreads();
        if (states && quarter == 0 && exists) states[(jl.i * tiles + tile) * p.U + jl.u + ch % S::V] = carry;
        float c = carry;
#pragma unroll
        for (int q = 0; q < kQuarters; ++q) {
            if (q == quarter) c = carry;
            carry = red[q][ch][0] * carry + red[q][ch][1];
        }
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            ab[quarter * S::kPart + s][ch][0] = c;
            c = pA[s] * c + pB[s];
        }
        __syncthreads();
        float now[S::V];
#pragma unroll
        for (int j = 0; j < S::V; ++j) now[j] = ab[seg][lane * S::V + j][0];
        T* out = h + (l.i * p.steps + t0) * p.U + l.u;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            Pack<T> v;
            const bool on = t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                now[j] = a[s][j] * now[j] + b[s][j];
                v.e[j] = (T)(on ? sigmoid((float)xo[s].e[j]) * now[j] : 0.0f);
            }
            store_pack(out + s * p.U, v, t0 + s < p.steps ? l.valid : 0);
        }
        __syncthreads();
    }
    if (chunk == p.chunks - 1 && quarter == 0 && exists) c_last[at] = carry;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void scan_bwd_kernel(ScanArgs p, const float* __restrict__ states,
                                                            const T* __restrict__ dh, int64_t dn, int64_t dt,
                                                            const float* __restrict__ d_last, T* __restrict__ dg,
                                                            float* __restrict__ d_c0) {
    using S = Shape<T>;
    __shared__ float ab[S::kSegs][kChannels][3];     // A, B and the gradient's B; then the states before and behind
    __shared__ float red[kQuarters][kChannels][3];
    float (*before)[kChannels][2] = reinterpret_cast<float (*)[kChannels][2]>(&red[0][0][0]);
    const int64_t blocks = (p.n * p.groups + S::kGroups - 1) / S::kGroups;
    const int64_t chunk = blockIdx.x / blocks, block = blockIdx.x - chunk * blocks;
    const int lane = threadIdx.x % S::kGroups, seg = threadIdx.x / S::kGroups;
    const Lane l = lane_of<T>(p, block * S::kGroups + lane);
    const T* g = static_cast<const T*>(p.gates) + l.i * p.gn + l.u;
    const T* dhp = dh + l.i * dn + l.u;
    const int ch = threadIdx.x % kChannels, quarter = threadIdx.x / kChannels;
    const Lane jl = lane_of<T>(p, block * S::kGroups + ch / S::V);
    const bool exists = ch % S::V < jl.valid;
    const int64_t at = jl.i * p.U + jl.u + ch % S::V;
    const int64_t tiles = (p.steps + kTile - 1) / kTile;
    float carry = exists && d_last ? d_last[at] : 0.0f;     // E behind the tile
    if (chunk < p.chunks - 1) {
        float A, B;
        chunks_before(p, at, p.chunks - 1, p.chunks - 1 - chunk, -1, quarter, before, ch, exists, A, B);
        carry = A * carry + B;
    }
    const int64_t first = chunk * p.chunk_tiles;
    const int64_t last = first + p.chunk_tiles < tiles ? first + p.chunk_tiles : tiles;
    for (int64_t tile = last - 1; tile >= first; --tile) {
        const int64_t t0 = tile * kTile + seg * S::kSteps;
        Pack<T> xf[S::kSteps], xz[S::kSteps], xo[S::kSteps], d[S::kSteps];
        float kp[S::kSteps];
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const int valid = t0 + s < l.len ? l.valid : 0;
            const T* q = g + (t0 + s) * p.gt;
            xf[s] = load_pack(q, valid);
            xz[s] = load_pack(q + p.U, valid);
            xo[s] = load_pack(q + 2 * p.U, valid);
            d[s] = load_pack(dhp + (t0 + s) * dt, dh ? valid : 0);
            kp[s] = t0 + s < l.len ? keep_of(p, l.i, t0 + s) : 1.0f;
        }
        const float start = exists ? states[(jl.i * tiles + tile) * p.U + jl.u + ch % S::V] : 0.0f;
        {
            float A[S::V], B[S::V], G[S::V];
#pragma unroll
            for (int j = 0; j < S::V; ++j) A[j] = 1.0f, B[j] = 0.0f, G[j] = 0.0f;
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s) {
                if (t0 + s >= l.len) continue;
#pragma unroll
                for (int j = 0; j < S::V; ++j) {
                    float f, m;
                    sigmoid_pair((float)xf[s].e[j], f, m);
                    const float a = f * kp[s];
                    B[j] = a * B[j] + m * (float)xz[s].e[j];
                    A[j] *= a;
                    // E at the segment's first step is the sum of a_0 .. a_s (o dh)_s
                    G[j] += A[j] * (sigmoid((float)xo[s].e[j]) * (float)d[s].e[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                float* e = ab[seg][lane * S::V + j];
                e[0] = A[j], e[1] = B[j], e[2] = G[j];
            }
        }
        __syncthreads();
        float pA[S::kPart], pB[S::kPart], pG[S::kPart], qA = 1.0f, qB = 0.0f, qG = 0.0f;
#pragma unroll
        for (int s = 0; s < S::kPart; ++s) {
            const float* e = ab[quarter * S::kPart + s][ch];
            pA[s] = e[0], pB[s] = e[1], pG[s] = e[2];
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
            ab[quarter * S::kPart + s][ch][0] = c;
            c = pA[s] * c + pB[s];
        }
#pragma unroll
        for (int s = S::kPart - 1; s >= 0; --s) {
            ab[quarter * S::kPart + s][ch][1] = E;
            E = pA[s] * E + pG[s];
        }
        __syncthreads();
        float now[S::V], back[S::V], cs[S::kSteps][S::V];
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
            now[j] = ab[seg][lane * S::V + j][0];
            back[j] = ab[seg][lane * S::V + j][1];
        }
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            const bool on = t0 + s < l.len;
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                float f, m;
                sigmoid_pair((float)xf[s].e[j], f, m);
                cs[s][j] = now[j] * kp[s];
                now[j] = on ? f * cs[s][j] + m * (float)xz[s].e[j] : now[j];
            }
        }
        T* out = dg + (l.i * p.steps + t0) * 3 * p.U + l.u;
#pragma unroll
        for (int s = S::kSteps - 1; s >= 0; --s) {
            const bool on = t0 + s < l.len;
            Pack<T> vf, vz, vo;
#pragma unroll
            for (int j = 0; j < S::V; ++j) {
                float f, m, o, om;
                sigmoid_pair((float)xf[s].e[j], f, m);
                sigmoid_pair((float)xo[s].e[j], o, om);
                const float z = (float)xz[s].e[j], dd = (float)d[s].e[j], pr = cs[s][j];
                const float cc = f * pr + m * z;
                const float od = o * dd;
                const float D = od + back[j];
                vf.e[j] = (T)(on ? D * (pr - z) * (f * m) : 0.0f);
                vz.e[j] = (T)(on ? D * m : 0.0f);
                vo.e[j] = (T)(on ? od * om * cc : 0.0f);
                back[j] = on ? f * kp[s] * D : back[j];
            }
            const int valid = t0 + s < p.steps ? l.valid : 0;
            T* w = out + s * 3 * p.U;
            store_pack(w, vf, valid);
            store_pack(w + p.U, vz, valid);
            store_pack(w + 2 * p.U, vo, valid);
        }
        __syncthreads();
    }
    if (d_c0 && chunk == 0 && quarter == 0 && exists) d_c0[at] = carry;
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
    sigmoid_pair((float)g[0], f, b);
    const float p = keep ? c[id] * keep[i] : c[id];
    const float now = f * p + b * (float)g[U];
    c_out[id] = now;
    h[id] = (T)(sigmoid((float)g[2 * U]) * now);
}

bool blocks_of(int64_t items, unsigned& blocks) {
    const int64_t b = (items + kThreads - 1) / kThreads;
    blocks = (unsigned)b;
    return b <= 0x7fffffff;
}

int64_t width_of(int32_t dtype) { return dtype == SWARM_F32 ? 4 : 8; }

// How the length is split: whole tiles, as many chunks as fill the card together with the channels.
void split(int64_t n, int64_t T, int64_t U, int64_t V, int64_t& groups, int64_t& blocks, int64_t& chunk_tiles,
           int64_t& chunks) {
    groups = (U + V - 1) / V;
    blocks = (n * groups + kChannels / V - 1) / (kChannels / V);
    const int64_t tiles = SWARM_GATED_TILES(T);
    int64_t want = blocks >= kFill ? 1 : (kFill + blocks - 1) / blocks;
    if (want > tiles) want = tiles;
    chunk_tiles = (tiles + want - 1) / want;
    chunks = (tiles + chunk_tiles - 1) / chunk_tiles;
}

}  // namespace

extern "C" {

int64_t swarm_gated_scan_workspace(int64_t n, int64_t T, int64_t U) {
    if (n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return 0;
    int64_t most = 0;
    for (int64_t V : {4, 8}) {
        int64_t groups, blocks, chunk_tiles, chunks;
        split(n, T, U, V, groups, blocks, chunk_tiles, chunks);
        if (chunks > most) most = chunks;
    }
    return most > 1 ? most * 2 * n * U : 0;
}

int32_t swarm_gated_scan_forward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                 int64_t gates_t, const float* c0, const float* keep, const int64_t* lengths, void* h,
                                 float* c_last, float* tile_states, float* work, void* stream) {
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    if (!gates || !h || !c_last || gates_t < 0 || gates_n < 0) return SWARM_ERR_ARG;
    ScanArgs p{n, T, U, gates, gates_n, gates_t, keep, lengths, 0, 0, 0, work};
    int64_t blocks;
    split(n, T, U, width_of(dtype), p.groups, blocks, p.chunk_tiles, p.chunks);
    if (blocks * p.chunks > 0x7fffffff || (p.chunks > 1 && !work)) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        if (p.chunks > 1)
            chunk_kernel<E, false><<<(unsigned)(blocks * (p.chunks - 1)), kThreads, 0, st>>>(p, nullptr, 0, 0);
        scan_fwd_kernel<E><<<(unsigned)(blocks * p.chunks), kThreads, 0, st>>>(p, c0, static_cast<E*>(h), c_last,
                                                                             tile_states);
    });
    return swarm::record_hip_status();
}

int32_t swarm_gated_scan_backward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                  int64_t gates_t, const float* keep, const int64_t* lengths,
                                  const float* tile_states, const void* d_h, int64_t d_h_n, int64_t d_h_t,
                                  const float* d_last, void* d_gates, float* d_c0, float* work, void* stream) {
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    if (!gates || !tile_states || !d_gates || gates_t < 0 || gates_n < 0 || d_h_n < 0 || d_h_t < 0)
        return SWARM_ERR_ARG;
    ScanArgs p{n, T, U, gates, gates_n, gates_t, keep, lengths, 0, 0, 0, work};
    int64_t blocks;
    split(n, T, U, width_of(dtype), p.groups, blocks, p.chunk_tiles, p.chunks);
    if (blocks * p.chunks > 0x7fffffff || (p.chunks > 1 && !work)) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const E* dh = static_cast<const E*>(d_h);
        if (p.chunks > 1)
            chunk_kernel<E, true><<<(unsigned)(blocks * (p.chunks - 1)), kThreads, 0, st>>>(p, dh, d_h_n, d_h_t);
        scan_bwd_kernel<E><<<(unsigned)(blocks * p.chunks), kThreads, 0, st>>>(p, tile_states, dh, d_h_n, d_h_t, d_last,
                                                                             static_cast<E*>(d_gates), d_c0);
    });
    return swarm::record_hip_status();
}

int32_t swarm_gated_step(int32_t dtype, int64_t rows, int64_t U, const void* gates, int64_t gates_row, const float* c,
                         const float* keep, void* h, float* c_out, void* stream) {
    if (!known_type(dtype) || rows < 0 || U < 1 || !sane(rows, U)) return SWARM_ERR_ARG;
    if (rows == 0) return SWARM_OK;
    unsigned blocks;
    if (!gates || !c || !h || !c_out || gates_row < 0 || !blocks_of(rows * U, blocks)) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        step_kernel<E><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            rows, U, static_cast<const E*>(gates), gates_row, c, keep, static_cast<E*>(h), c_out);
    });
    return swarm::record_hip_status();
}

}  // extern "C"
