// Embedding lookup and its gradient.
//
// lookup: out[t] = scale * table[id_t], one group of lanes per row; bound by the bytes of the rows
// read and written.
//
// gradient: out[v] (+)= scale * sum_{t: id_t = v} grad[t]. The ids are sorted (stable, so that equal ids
// keep the order of t), cut into pieces of 32 positions, and each warp sums the runs of one piece over one
// span of columns. A run inside a piece is written at once; a run that crosses a border leaves one partial
// sum for each piece, and a second kernel adds those in order. No float is added by an atomic, so the sums
// have one order, which the ids alone fix.
#include "tb_encoder.h"
#include "tb_vec.cuh"

namespace tb {

namespace {

__device__ __forceinline__ int64_t load_id(const void* ids, int id64, int64_t t) {
    return id64 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
}

// id -> row in [0, V), or -1; an id that is neither -1 nor a row is reported.
__device__ __forceinline__ int32_t valid_row(int64_t id, int64_t V, int32_t* status) {
    if (id >= 0 && id < V) return (int32_t)id;
    if (id != -1 && status) atomicOr(status, TRIDENT_STATUS_BAD_ID);
    return -1;
}

// ---- lookup

template <class T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ table, int64_t V, int n, int64_t ld,
                                                     const void* __restrict__ ids, int id64, int64_t count, float scale,
                                                     T* __restrict__ out, int64_t ld_out, int32_t* status, int log_lanes) {
    const int lane = threadIdx.x & ((1 << log_lanes) - 1);
    const int64_t t = (int64_t)blockIdx.x * (256 >> log_lanes) + (threadIdx.x >> log_lanes);
    if (t >= count) return;
    const int64_t id = load_id(ids, id64, t);
    T* o = out + t * ld_out;
    const int step = 1 << log_lanes;
    if (id < 0 || id >= V) {
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = id == -1 ? 0.0f : __int_as_float(0x7fffffff);
        const Pack<T, VEC> p = Pack<T, VEC>::of(f);
        for (int v = lane; v < n; v += step) p.store(o + (int64_t)v * VEC);
        if (id != -1 && status && lane == 0) atomicOr(status, TRIDENT_STATUS_BAD_ID);
        return;
    }
    const T* row = table + id * ld;
    for (int v = lane; v < n; v += 4 * step) {
        Pack<T, VEC> p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (v + k * step < n) p[k] = Pack<T, VEC>::load(row + (int64_t)(v + k * step) * VEC);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (v + k * step >= n) break;
            float f[VEC];
            p[k].get(f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] *= scale;
            Pack<T, VEC>::of(f).store(o + (int64_t)(v + k * step) * VEC);
        }
    }
}

template <class T>
cudaError_t lookup(const T* table, int64_t V, int D, int64_t ld, const void* ids, int id64, int64_t count, float scale,
                   T* out, int64_t ld_out, int32_t* status, cudaStream_t st) {
    constexpr int kMax = 16 / (int)sizeof(T);
    const int vec = wide_elements({{table, ld, (int)sizeof(T)}, {out, ld_out, (int)sizeof(T)}}, D, kMax);
    const int n = D / vec;
    int log_lanes = 0;
    while (log_lanes < 5 && (1 << log_lanes) < n) ++log_lanes;
    const int64_t grid = (count + (256 >> log_lanes) - 1) / (256 >> log_lanes);
    auto go = [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        lookup_kernel<T, VEC><<<(unsigned)grid, 256, 0, st>>>(table, V, n, ld, ids, id64, count, scale, out, ld_out,
                                                             status, log_lanes);
    };
    with_vec<kMax>(vec, go);
    return cudaGetLastError();
}

// ---- gradient: few ids, without a sort

constexpr int kDirectIds = 1024;

// One block per position t. The block of an id's first occurrence collects the positions of all of them in
// order and sums their rows; the others leave. No run is long here (<= 1024 rows, over 8 warps).
template <class T, class O, int VEC>
__global__ void __launch_bounds__(256) grad_direct_kernel(const T* __restrict__ grad, int64_t ld, const void* __restrict__ ids,
                                                          int id64, int count, int64_t V, int n, float scale, int accumulate,
                                                          O* __restrict__ out, int64_t ld_out, int32_t* status) {
    __shared__ int32_t list[kDirectIds];
    __shared__ int warp_count[8];
    __shared__ __align__(16) float part[8][32 * VEC];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t row = valid_row(load_id(ids, id64, t), V, threadIdx.x == 0 ? status : nullptr);
    if (row < 0) return;
    // thread i looks at positions 4 i .. 4 i + 3: a warp's positions are consecutive
    bool hit[4];
    bool earlier = false;
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int j = threadIdx.x * 4 + k;
        hit[k] = j < count && load_id(ids, id64, j) == row;
        earlier |= hit[k] && j < t;
        mine += hit[k];
    }
    if (__syncthreads_or(earlier)) return;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    if (lane == 31) warp_count[warp] = before;
    before -= mine;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) before += warp_count[w];
        total += warp_count[w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (hit[k]) list[before++] = threadIdx.x * 4 + k;
    __syncthreads();
    O* o = out + (int64_t)row * ld_out;
    auto finish = [&](int v, float* acc) {
        float old[VEC];
        if (accumulate) load_n<O, VEC>(o + (int64_t)v * VEC, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = accumulate ? fmaf(acc[i], scale, old[i]) : acc[i] * scale;
        store_n<O, VEC>(o + (int64_t)v * VEC, acc);
    };
    if (total <= 8) {
        for (int v = threadIdx.x; v < n; v += 256) {
            float acc[VEC] = {};
            for (int j = 0; j < total; ++j) {
                float f[VEC];
                Pack<T, VEC>::load(grad + (int64_t)list[j] * ld + (int64_t)v * VEC).get(f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += f[i];
            }
            finish(v, acc);
        }
        return;
    }
    // warp w sums an eighth of the list (consecutive positions), then the eighths are added in order
    const int lo = total * warp / 8, hi = total * (warp + 1) / 8;
    for (int v0 = 0; v0 < n; v0 += 32) {
        const int v = v0 + lane;
        float acc[VEC] = {};
        if (v < n) {
#pragma unroll 8
            for (int j = lo; j < hi; ++j) {
                float f[VEC];
                Pack<T, VEC>::load(grad + (int64_t)list[j] * ld + (int64_t)v * VEC).get(f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += f[i];
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[warp][lane * VEC + i] = acc[i];
        __syncthreads();
        if (warp == 0 && v < n) {
#pragma unroll
            for (int w = 1; w < 8; ++w)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += part[w][lane * VEC + i];
            finish(v, acc);
        }
        __syncthreads();
    }
}

// ---- gradient: stable radix sort of (id, position)

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBins = 512;              // 9 bits a pass: two passes sort ids below 2^18
constexpr int kSubTile = kSortThreads * 4;
constexpr int kMaxTiles = 256;             // blocks of a pass; each reads the counts of all

struct SortPass {
    const void* ids;       // pass 0
    int id64;
    int64_t V;
    const int32_t* keys;   // later passes
    const int32_t* pos;
    int32_t* n_valid;
    int64_t count;
    int64_t tile;          // positions of a block, a multiple of kSubTile
    int shift, bits, first;
};

// counts[block][digit] of the block's valid keys.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass s, int32_t* __restrict__ counts, int32_t* status) {
    __shared__ int32_t hist[kMaxBins];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t n = s.first ? s.count : (int64_t)*s.n_valid;
    const int64_t lo = (int64_t)blockIdx.x * s.tile, hi = min(n, lo + s.tile);
    const int mask = (1 << s.bits) - 1;
    for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
        const int32_t key = s.first ? valid_row(load_id(s.ids, s.id64, i), s.V, status) : s.keys[i];
        if (key >= 0) atomicAdd(&hist[(key >> s.shift) & mask], 1);
    }
    __syncthreads();
    if (threadIdx.x <= mask) counts[(int64_t)blockIdx.x * kMaxBins + threadIdx.x] = hist[threadIdx.x];
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortPass s, const int32_t* __restrict__ counts, int tiles,
                                                                    int32_t* __restrict__ keys_out, int32_t* __restrict__ pos_out) {
    __shared__ int32_t warp_hist[kSortWarps][kMaxBins];
    __shared__ int32_t offset[kMaxBins];
    __shared__ int32_t scan[kSortWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int mask = (1 << s.bits) - 1;
    // where this block's keys of digit `tid` go: after all smaller digits, and this digit's in earlier blocks
    int total = 0, before = 0;
    if (tid <= mask) {
#pragma unroll 8
        for (int b = 0; b < tiles; ++b) {
            const int c = counts[(int64_t)b * kMaxBins + tid];
            total += c;
            if (b < (int)blockIdx.x) before += c;
        }
    }
    int incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int base = incl - total;
    int all = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        if (w < warp) base += scan[w];
        all += scan[w];
    }
    offset[tid] = base + before;
    if (s.first && blockIdx.x == 0 && tid == 0) *s.n_valid = all;
    const int64_t n = s.first ? s.count : (int64_t)all;
    const int64_t lo = (int64_t)blockIdx.x * s.tile, hi = min(n, lo + s.tile);
    for (int64_t sub = lo; sub < hi; sub += kSubTile) {
        for (int i = lane; i <= mask; i += 32) warp_hist[warp][i] = 0;
        __syncwarp();
        int32_t key[4], pos[4], rank[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // a warp's 128 positions are consecutive
            const int64_t i = sub + warp * 128 + k * 32 + lane;
            key[k] = -1;
            if (i < hi) {
                key[k] = s.first ? valid_row(load_id(s.ids, s.id64, i), s.V, nullptr) : s.keys[i];
                pos[k] = s.first ? (int32_t)i : s.pos[i];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int digit = (key[k] >> s.shift) & mask;
            const unsigned valid = __ballot_sync(0xffffffffu, key[k] >= 0);
            unsigned same = valid;  // lanes with this lane's digit
            for (int b = 0; b < s.bits; ++b) {
                const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1);
                same &= ((digit >> b) & 1) ? set : ~set;
            }
            const unsigned lower = same & ((1u << lane) - 1);
            int prior = 0;
            if (key[k] >= 0) prior = warp_hist[warp][digit];
            __syncwarp();
            if (key[k] >= 0 && lower == 0) warp_hist[warp][digit] = prior + __popc(same);
            __syncwarp();
            rank[k] = prior + __popc(lower);
        }
        __syncthreads();
        if (tid <= mask) {
            int at = offset[tid];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = warp_hist[w][tid];
                warp_hist[w][tid] = at;
                at += c;
            }
            offset[tid] = at;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (key[k] < 0) continue;
            const int dst = warp_hist[warp][(key[k] >> s.shift) & mask] + rank[k];
            keys_out[dst] = key[k];
            pos_out[dst] = pos[k];
        }
        __syncthreads();
    }
}

// ---- gradient: sums of the sorted runs

constexpr int kPiece = 32;

struct RunArgs {
    const int32_t* keys;
    const int32_t* pos;
    const int32_t* n_valid;
    float* part;         // [pieces][2][ld_part]: a run from the piece before, a run into the next
    int64_t ld_part;
    int64_t ld, ld_out;
    int cols;            // wide columns (D / VEC)
    int spans;           // ceil(cols / 32)
    float scale;
    int accumulate;
};

template <class O, int VEC>
__device__ __forceinline__ void finish_row(const RunArgs& a, O* out, int32_t key, int v, float* acc) {
    O* o = out + (int64_t)key * a.ld_out + (int64_t)v * VEC;
    if (a.accumulate) {
        float old[VEC];
        load_n<O, VEC>(o, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(acc[i], a.scale, old[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
    }
    store_n<O, VEC>(o, acc);
}

template <class T, class O, int VEC>
__global__ void __launch_bounds__(256) run_sum_kernel(RunArgs a, const T* __restrict__ grad, O* __restrict__ out) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t piece = unit / a.spans;
    const int v = (int)(unit % a.spans) * 32 + lane;
    const int n = *a.n_valid;
    const int64_t first = piece * kPiece;
    if (first >= n) return;
    const int m = (int)min((int64_t)kPiece, n - first);
    const int32_t key = lane < m ? a.keys[first + lane] : -1;
    const int32_t pos = lane < m ? a.pos[first + lane] : 0;
    const int32_t prev = first > 0 ? a.keys[first - 1] : -1;
    const int32_t next = first + m < n ? a.keys[first + m] : -1;
    const bool on = v < a.cols;
    const T* col = grad + (int64_t)v * VEC;
    float acc[VEC] = {};
    int start = 0;
    for (int j0 = 0; j0 < m; j0 += 8) {
        Pack<T, VEC> p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int32_t r = __shfl_sync(0xffffffffu, pos, j0 + k);
            if (on && j0 + k < m) p[k] = Pack<T, VEC>::load_stream(col + (int64_t)r * a.ld);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int j = j0 + k;
            const int32_t kj = __shfl_sync(0xffffffffu, key, j);
            const int32_t after = __shfl_sync(0xffffffffu, key, (j + 1) & 31);
            if (j >= m) continue;
            if (on) {
                float f[VEC];
                p[k].get(f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += f[i];
            }
            const bool last = j + 1 == m;
            if (last || after != kj) {
                const bool from_before = start == 0 && prev == kj;
                const bool into_next = last && next == kj;
                if (on) {
                    if (from_before || into_next) {
                        float* slot = a.part + (piece * 2 + (from_before ? 0 : 1)) * a.ld_part + (int64_t)v * VEC;
                        store_n<float, VEC>(slot, acc);
                    } else {
                        finish_row<O, VEC>(a, out, kj, v, acc);
                    }
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
                start = j + 1;
            }
        }
    }
}

constexpr int kJoinAlone = 16;  // partial sums that one warp adds by itself

// Adds the partial sums of each run that crosses pieces: slot 1 of its first piece, then slot 0 of the
// others, in order. One warp per (piece, span); a long run is shared by the block's 8 warps.
template <class O, int VEC>
__global__ void __launch_bounds__(256) run_join_kernel(RunArgs a, O* __restrict__ out) {
    __shared__ int64_t long_first[8], long_last[8];
    __shared__ int32_t long_key[8];
    __shared__ __align__(16) float sums[8][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t group = blockIdx.x / a.spans;
    const int v = (int)(blockIdx.x % a.spans) * 32 + lane;
    const bool on = v < a.cols;
    const int64_t piece = group * 8 + warp;
    const int n = *a.n_valid;
    auto add = [&](float* acc, int64_t lo, int64_t hi) {  // slot 0 of pieces [lo, hi)
#pragma unroll 4
        for (int64_t q = lo; q < hi; ++q) {
            float f[VEC];
            load_n<float, VEC>(a.part + q * 2 * a.ld_part + (int64_t)v * VEC, f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += f[i];
        }
    };
    bool is_long = false;
    const int64_t end = (piece + 1) * kPiece;
    if (end < n) {
        const int32_t key = a.keys[end - 1];
        const bool crosses = a.keys[end] == key;
        const bool begins = a.keys[end - kPiece] != key || piece == 0 || a.keys[end - kPiece - 1] != key;
        if (crosses && begins) {
            int64_t lo = end, hi = n;  // the run's end: the first position of a larger key
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (a.keys[mid] == key) lo = mid + 1; else hi = mid;
            }
            const int64_t last = (lo - 1) / kPiece;
            if (last - piece < kJoinAlone) {
                if (on) {
                    float acc[VEC];
                    load_n<float, VEC>(a.part + (piece * 2 + 1) * a.ld_part + (int64_t)v * VEC, acc);
                    add(acc, piece + 1, last + 1);
                    finish_row<O, VEC>(a, out, key, v, acc);
                }
            } else {
                is_long = true;
                if (lane == 0) {
                    long_first[warp] = piece;
                    long_last[warp] = last;
                    long_key[warp] = key;
                }
            }
        }
    }
    if (lane == 0 && !is_long) long_key[warp] = -1;
    __syncthreads();
    for (int r = 0; r < 8; ++r) {
        if (long_key[r] < 0) continue;
        const int64_t lo = long_first[r] + 1, m = long_last[r] + 1 - lo;
        float acc[VEC] = {};
        if (on) {
            if (warp == 0) load_n<float, VEC>(a.part + (long_first[r] * 2 + 1) * a.ld_part + (int64_t)v * VEC, acc);
            add(acc, lo + m * warp / 8, lo + m * (warp + 1) / 8);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sums[warp][lane * VEC + i] = acc[i];
        __syncthreads();
        if (warp == 0 && on) {
#pragma unroll
            for (int w = 1; w < 8; ++w)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += sums[w][lane * VEC + i];
            finish_row<O, VEC>(a, out, long_key[r], v, acc);
        }
        __syncthreads();
    }
}

struct GradWorkspace {
    int32_t* n_valid;
    int32_t* counts;     // [kMaxTiles][kMaxBins]
    int32_t* keys[2];
    int32_t* pos[2];
    float* part;
};

int64_t part_stride(int D) { return (D + 3) / 4 * 4; }

size_t carve_grad(int64_t T, int D, void* base, GradWorkspace* ws) {
    size_t off = 0;
    char* p = static_cast<char*>(base);
    auto take = [&](size_t bytes) -> void* {
        void* r = p ? (void*)(p + off) : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return r;
    };
    GradWorkspace w;
    w.n_valid = (int32_t*)take(256);
    if (T > kDirectIds) {
        w.counts = (int32_t*)take((size_t)kMaxTiles * kMaxBins * 4);
        for (int i = 0; i < 2; ++i) w.keys[i] = (int32_t*)take((size_t)T * 4);
        for (int i = 0; i < 2; ++i) w.pos[i] = (int32_t*)take((size_t)T * 4);
        w.part = (float*)take((size_t)((T + kPiece - 1) / kPiece) * 2 * part_stride(D) * 4);
    }
    if (ws) *ws = w;
    return off;
}

template <class T, class O>
cudaError_t grad_typed(const T* grad, int64_t ld, const void* ids, int id64, int64_t count, int64_t V, int D, float scale,
                       int accumulate, O* out, int64_t ld_out, void* workspace, int32_t* status, int* launches,
                       cudaStream_t st) {
    cudaError_t e;
    if (!accumulate) {
        e = ld_out == D ? cudaMemsetAsync(out, 0, (size_t)V * D * sizeof(O), st)
                        : cudaMemset2DAsync(out, ld_out * sizeof(O), 0, (size_t)D * sizeof(O), V, st);
        if (e != cudaSuccess) return e;
    }
    if (count == 0) return cudaSuccess;
    constexpr int kMax = 16 / (int)sizeof(T);
    int vec = wide_elements({{grad, ld, (int)sizeof(T)}, {out, ld_out, (int)sizeof(O)}}, D, kMax);
    if (count <= kDirectIds) {
        with_vec<kMax>(vec, [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            grad_direct_kernel<T, O, VEC><<<(unsigned)count, 256, 0, st>>>(grad, ld, ids, id64, (int)count, V, D / vec,
                                                                          scale, accumulate, out, ld_out, status);
        });
        *launches += 1;
        return cudaGetLastError();
    }
    GradWorkspace ws;
    carve_grad(count, D, workspace, &ws);
    int bits = 1;
    while (bits < 31 && ((int64_t)1 << bits) < V) ++bits;
    const int passes = (bits + 8) / 9;
    SortPass s;
    s.ids = ids;
    s.id64 = id64;
    s.V = V;
    s.n_valid = ws.n_valid;
    s.count = count;
    s.bits = (bits + passes - 1) / passes;
    s.tile = ((count + kMaxTiles - 1) / kMaxTiles + kSubTile - 1) / kSubTile * kSubTile;
    const int tiles = (int)((count + s.tile - 1) / s.tile);
    for (int p = 0; p < passes; ++p) {
        s.first = p == 0;
        s.shift = p * s.bits;
        s.keys = ws.keys[(p + 1) & 1];
        s.pos = ws.pos[(p + 1) & 1];
        sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(s, ws.counts, status);
        sort_scatter_kernel<<<tiles, kSortThreads, 0, st>>>(s, ws.counts, tiles, ws.keys[p & 1], ws.pos[p & 1]);
    }
    RunArgs a;
    a.keys = ws.keys[(passes - 1) & 1];
    a.pos = ws.pos[(passes - 1) & 1];
    a.n_valid = ws.n_valid;
    a.part = ws.part;
    a.ld_part = part_stride(D);
    a.ld = ld;
    a.ld_out = ld_out;
    a.scale = scale;
    a.accumulate = accumulate;
    while (vec > 1 && D / vec < 32) vec /= 2;  // a narrow row over all lanes of a warp
    a.cols = D / vec;
    a.spans = (a.cols + 31) / 32;
    const int64_t pieces = (count + kPiece - 1) / kPiece;
    const int64_t grid = (pieces * a.spans + 7) / 8, join_grid = (pieces + 7) / 8 * a.spans;
    if (grid > 0x7fffffff || join_grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    with_vec<kMax>(vec, [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        run_sum_kernel<T, O, VEC><<<(unsigned)grid, 256, 0, st>>>(a, grad, out);
        run_join_kernel<O, VEC><<<(unsigned)join_grid, 256, 0, st>>>(a, out);
    });
    *launches += 2 * passes + 2;
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_embed_lookup(const void* table, int dtype, int64_t V, int D, int64_t ld, const void* ids, int id64,
                                int64_t count, float scale, void* out, int64_t ld_out, int32_t* status, cudaStream_t st) {
    return with_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        return lookup<T>(static_cast<const T*>(table), V, D, ld, ids, id64, count, scale, static_cast<T*>(out), ld_out,
                         status, st);
    });
}

size_t embed_grad_workspace(int64_t T, int D) { return carve_grad(T, D, nullptr, nullptr); }

cudaError_t launch_embed_grad(const void* grad, int dtype, int64_t ld, const void* ids, int id64, int64_t count, int64_t V,
                              int D, float scale, int accumulate, void* out, int out_dtype, int64_t ld_out,
                              void* workspace, int32_t* status, int* launches, cudaStream_t st) {
    return with_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        const T* g = static_cast<const T*>(grad);
        if (out_dtype == TRIDENT_F32)
            return grad_typed<T, float>(g, ld, ids, id64, count, V, D, scale, accumulate, static_cast<float*>(out), ld_out,
                                        workspace, status, launches, st);
        return grad_typed<T, T>(g, ld, ids, id64, count, V, D, scale, accumulate, static_cast<T*>(out), ld_out, workspace,
                                status, launches, st);
    });
}

}  // namespace tb
