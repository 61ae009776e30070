// Embedding lookup and its gradient.
//
// lookup: out[t] = scale * table[id_t], one group of lanes per row; bound by the bytes of the rows
// read and written: 320,000 ids (a fifth of them -1) of 960 bf16 columns take 120 us on a B200, 5.7 TB/s.
// Small lookups are bound by their call (9 us of host time, of which 4 are the launch).
//
// gradient: out[v] (+)= scale * sum_{t: id_t = v} grad[t]. The ids are sorted (stable, so that equal ids
// keep the order of t), cut into pieces of 32 positions, and each warp sums the runs of one piece over one
// span of columns. A run inside a piece is written at once; a run that crosses a border leaves one partial
// sum for each piece, and a second kernel adds those in a fixed order. So every sum has one order, which the
// ids alone fix, and frequent ids are shared by many warps. Zeros of a table that is written whole go out on a
// second stream while the ids are sorted.
//
// 32,000 ids into 65,536 x 960 bf16 rows take 47 us (28 us of bytes): the sort 16 us beside 20 us of zeros,
// the sums 17, the joins 6. 320,000 ids added to a 262,144 x 128 float32 table take 63 us (20 us of bytes): the
// sort's four launches 28 us, the sums 22, the joins 9. Both are bound by the latency of the steps, not by
// memory.
#include <cooperative_groups.h>

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

// A group of lanes takes ROWS rows, whose loads are all under way before the first is stored.
template <class T, int VEC, int ROWS>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ table, int64_t V, int n, int64_t ld,
                                                     const void* __restrict__ ids, int id64, int64_t count, float scale,
                                                     T* __restrict__ out, int64_t ld_out, int32_t* status, int log_lanes) {
    const int lane = threadIdx.x & ((1 << log_lanes) - 1);
    const int64_t t0 = ((int64_t)blockIdx.x * (256 >> log_lanes) + (threadIdx.x >> log_lanes)) * ROWS;
    const int step = 1 << log_lanes;
    int64_t id[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) id[r] = t0 + r < count ? load_id(ids, id64, t0 + r) : -1;
    // where row r comes from: a row of the table, or a value in its place
    bool there[ROWS];
    float other[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        there[r] = id[r] >= 0 && id[r] < V;
        other[r] = id[r] == -1 ? 0.0f : __int_as_float(0x7fffffff);
        if (!there[r] && id[r] != -1 && status && lane == 0) atomicOr(status, TRIDENT_STATUS_BAD_ID);
    }
    for (int v = lane; v < n; v += 4 * step) {
        Pack<T, VEC> p[ROWS][4];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (there[r] && v + k * step < n) p[r][k] = Pack<T, VEC>::load(table + id[r] * ld + (int64_t)(v + k * step) * VEC);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (t0 + r >= count) break;
            T* o = out + (t0 + r) * ld_out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (v + k * step >= n) break;
                float f[VEC];
                if (there[r]) {
                    p[r][k].get(f);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[i] *= scale;
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[i] = other[r];
                }
                Pack<T, VEC>::of(f).store(o + (int64_t)(v + k * step) * VEC);
            }
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
    const int64_t per_block = 256 >> log_lanes;
    auto go = [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        auto with = [&](auto r) {
            constexpr int ROWS = decltype(r)::value;
            const int64_t grid = (count + per_block * ROWS - 1) / (per_block * ROWS);
            lookup_kernel<T, VEC, ROWS><<<(unsigned)grid, 256, 0, st>>>(table, V, n, ld, ids, id64, count, scale, out, ld_out,
                                                                       status, log_lanes);
        };
        // two rows at a time where a row gives a lane few bytes: 1,000,000 x 128 bf16 100 us (one at a time 112), 300,000 x
        // 97 bf16 57 us (70), 100,000 x 1001 float32 127 us (133); of 320,000 x 960 bf16 a lane has four 16-byte
        // columns already, 126 us (two at a time 129)
        if (count >= per_block * num_sms() * 8 && !(VEC * sizeof(T) == 16 && n > 64)) with(std::integral_constant<int, 2>{});
        else with(std::integral_constant<int, 1>{});
    };
    with_vec<kMax>(vec, go);
    return cudaGetLastError();
}

// ---- gradient: few ids, without a sort

// Up to this many ids: 256 and 1,024 ids of 960 bf16 columns take 8.5 and 10 us (the sort's three launches 24 and
// 27 us). At worst, 1,024 of two ids, two blocks read all rows, 36 us (18).
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
        for (int j0 = lo; j0 < hi && v < n; j0 += 16) {
            Pack<T, VEC> p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (j0 + k < hi) p[k] = Pack<T, VEC>::load(grad + (int64_t)list[j0 + k] * ld + (int64_t)v * VEC);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (j0 + k >= hi) break;
                float f[VEC];
                p[k].get(f);
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
//
// Two launches a pass of up to 9 bits: the counts of each block's keys, then the keys to their places. A block
// finds its places by adding up the counts of all blocks itself (at most kMaxTiles rows of 2 KB), which takes
// the time of a few loads in flight and spares a launch.

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBins = 512;              // 9 bits a pass: two passes sort ids below 2^18
constexpr int kSortKeys = 4;               // keys of a thread in a turn
constexpr int kSubTile = kSortThreads * kSortKeys;
constexpr int kMaxTiles = 256;             // blocks of a pass; each reads the counts of all

struct SortPass {
    const void* ids;       // pass 0
    int id64;
    int64_t V;
    const int2* in;        // later passes: (key, position)
    int2* out;
    int32_t* n_valid;
    int64_t count;
    int64_t tile;          // positions of a block, a multiple of kSubTile
    int shift, bits, first;
};

// counts[block][digit] of the block's valid keys.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass s, int32_t* __restrict__ counts, int32_t* status) {
    __shared__ int32_t hist[kMaxBins];
    wait_for_previous();
    if (threadIdx.x < kMaxBins) hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t n = s.first ? s.count : (int64_t)*s.n_valid;
    const int64_t lo = (int64_t)blockIdx.x * s.tile, hi = min(n, lo + s.tile);
    const int mask = (1 << s.bits) - 1;
    for (int64_t sub = lo; sub < hi; sub += kSubTile) {
        int32_t key[kSortKeys];
#pragma unroll
        for (int k = 0; k < kSortKeys; ++k) {
            const int64_t i = sub + k * kSortThreads + threadIdx.x;
            key[k] = -1;
            if (i < hi) key[k] = s.first ? valid_row(load_id(s.ids, s.id64, i), s.V, status) : s.in[i].x;
        }
#pragma unroll
        for (int k = 0; k < kSortKeys; ++k)
            if (key[k] >= 0) atomicAdd(&hist[(key[k] >> s.shift) & mask], 1);
    }
    __syncthreads();
    if (threadIdx.x <= mask) counts[(int64_t)blockIdx.x * kMaxBins + threadIdx.x] = hist[threadIdx.x];
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortPass s, const int32_t* __restrict__ counts, int tiles) {
    extern __shared__ __align__(16) int32_t warp_hist[];  // [kSortWarps][kMaxBins], then the turn's items in order
    __shared__ int32_t offset[kMaxBins];   // where the block's next key of a digit goes
    __shared__ int32_t start[kMaxBins];    // ... and its first of this turn in `sorted`
    __shared__ __align__(16) int32_t sums[2][kSortThreads * 4 / kMaxBins][kMaxBins];
    __shared__ int32_t scan[2][kMaxBins / 32];
    int2* sorted = reinterpret_cast<int2*>(warp_hist + kSortWarps * kMaxBins);
    wait_for_previous();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int mask = (1 << s.bits) - 1;
    // the first turn's keys are on their way meanwhile
    int2 item[kSortKeys];
    const int64_t most = s.count;  // (the later passes' arrays are as long; what is past n is not used)
    const int64_t lo = (int64_t)blockIdx.x * s.tile;
    auto load = [&](int64_t sub) {
#pragma unroll
        for (int k = 0; k < kSortKeys; ++k) {  // a warp's keys of a turn are consecutive
            const int64_t i = sub + warp * (32 * kSortKeys) + k * 32 + lane;
            item[k] = make_int2(-1, (int)i);
            if (i < most) {
                if (s.first) item[k].x = valid_row(load_id(s.ids, s.id64, i), s.V, nullptr);
                else item[k] = s.in[i];
            }
        }
    };
    load(lo);
    // where this block's keys of a digit go: after all smaller digits, and this digit's in earlier blocks.
    // Four digits a thread; the rows of counts are shared by kParts sets of threads.
    constexpr int kQuads = kMaxBins / 4, kParts = kSortThreads / kQuads;
    {
        int4 total = make_int4(0, 0, 0, 0), before = total;
        const int quad = tid & (kQuads - 1), part = tid / kQuads;
        if (quad * 4 <= mask) {
#pragma unroll 8
            for (int b = part; b < tiles; b += kParts) {
                const int4 c = *reinterpret_cast<const int4*>(counts + (int64_t)b * kMaxBins + quad * 4);
                total.x += c.x; total.y += c.y; total.z += c.z; total.w += c.w;
                if (b < (int)blockIdx.x) { before.x += c.x; before.y += c.y; before.z += c.z; before.w += c.w; }
            }
        }
        *reinterpret_cast<int4*>(&sums[0][part][quad * 4]) = total;
        *reinterpret_cast<int4*>(&sums[1][part][quad * 4]) = before;
    }
    __syncthreads();
    // exclusive sum over the digits of one value a digit, by the first kMaxBins threads; `all`: their sum
    auto scan_bins = [&](int value, int which, int& all) {
        int incl = value;
        if (tid < kMaxBins) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            if (lane == 31) scan[which][warp] = incl;
        }
        __syncthreads();
        int base = incl - value;
        all = 0;
#pragma unroll
        for (int w = 0; w < kMaxBins / 32; ++w) {
            const int c = scan[which][w];
            if (w < warp) base += c;
            all += c;
        }
        return base;
    };
    int total = 0, before = 0, all;
    if (tid <= mask) {
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
            total += sums[0][q][tid];
            before += sums[1][q][tid];
        }
    }
    const int base = scan_bins(total, 0, all);
    if (tid < kMaxBins) offset[tid] = base + before;
    if (s.first && blockIdx.x == 0 && tid == 0) *s.n_valid = all;
    const int64_t n = s.first ? s.count : (int64_t)all, hi = min(n, lo + s.tile);
    int32_t* mine = warp_hist + warp * kMaxBins;
    for (int64_t sub = lo; sub < hi; sub += kSubTile) {
        if (sub > lo) load(sub);
        for (int i = lane; i <= mask; i += 32) mine[i] = 0;
        __syncwarp();
        int32_t rank[kSortKeys];
#pragma unroll
        for (int k = 0; k < kSortKeys; ++k) {
            if (sub + warp * (32 * kSortKeys) + k * 32 + lane >= hi) item[k].x = -1;
            const int digit = (item[k].x >> s.shift) & mask;
            unsigned same = __ballot_sync(0xffffffffu, item[k].x >= 0);  // lanes with this lane's digit
            for (int b = 0; b < s.bits; ++b) {
                const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1);
                same &= ((digit >> b) & 1) ? set : ~set;
            }
            const unsigned lower = same & ((1u << lane) - 1);
            int prior = 0;
            if (item[k].x >= 0) prior = mine[digit];
            __syncwarp();
            if (item[k].x >= 0 && lower == 0) mine[digit] = prior + __popc(same);
            __syncwarp();
            rank[k] = prior + __popc(lower);
        }
        __syncthreads();
        int count = 0, turn;
        if (tid <= mask) {
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = warp_hist[w * kMaxBins + tid];
                warp_hist[w * kMaxBins + tid] = count;
                count += c;
            }
        }
        const int first = scan_bins(count, 1, turn);
        if (tid < kMaxBins) start[tid] = first;
        __syncthreads();
        // in order in shared memory first: the keys of a digit then leave together
#pragma unroll
        for (int k = 0; k < kSortKeys; ++k) {
            const int digit = (item[k].x >> s.shift) & mask;
            if (item[k].x >= 0) sorted[start[digit] + mine[digit] + rank[k]] = item[k];
        }
        __syncthreads();
        for (int i = tid; i < turn; i += kSortThreads) {
            const int2 it = sorted[i];
            const int digit = (it.x >> s.shift) & mask;
            s.out[offset[digit] + i - start[digit]] = it;
        }
        __syncthreads();
        if (tid <= mask) offset[tid] += count;
        __syncthreads();
    }
}

// The whole sort in one launch, for up to kClusterIds ids: a cluster of kClusterBlocks thread blocks, whose
// barriers stand where the launches above part. Each warp owns a run of positions: it counts its digits, the
// counts are added up over the block's warps and then over the cluster's blocks (read from their shared
// memory), and the warp goes over its keys again in order. More ids than that are written out faster by more
// SMs than a cluster has. The whole gradient of 8 columns with ids below 65,536 takes, with this and with
// separate launches: 31 and 41 us for 32,000 ids, 48 and 46 us for 131,000, 83 and 59 us for 320,000.
constexpr int kClusterBlocks = 16;
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int64_t kClusterIds = 131072;
constexpr int kClusterSmem = (kClusterWarps + 2) * kMaxBins * 4;

struct ClusterSort {
    const void* ids;
    int id64;
    int64_t V;
    int count, bits, passes;
    int2* items[2];
    int32_t *n_valid, *status;
};

__global__ void __launch_bounds__(kClusterThreads) sort_cluster_kernel(ClusterSort s) {
    extern __shared__ int32_t sh[];
    __shared__ int32_t scan[kClusterWarps];
    wait_for_previous();
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int32_t* mine = sh + warp * kMaxBins;            // this warp's counts, then where its next key of a digit goes
    int32_t* total = sh + kClusterWarps * kMaxBins;  // the block's counts
    int32_t* offset = total + kMaxBins;
    const int rank = (int)cluster.block_rank();
    const int bins = 1 << s.bits;
    const int seg = ((s.count + kClusterBlocks * kClusterWarps - 1) / (kClusterBlocks * kClusterWarps) + 31) / 32 * 32;
    const int lo = (rank * kClusterWarps + warp) * seg;
    int n = s.count;
    for (int p = 0; p < s.passes; ++p) {
        const int shift = p * s.bits;
        const int2* in = s.items[(p + 1) & 1];
        int2* out = s.items[p & 1];
        const int hi = min(n, lo + seg);
        auto load = [&](int i0, int2* item, int32_t* status) {  // kSortKeys rounds of 32 at a time
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k) {
                const int i = i0 + k * 32 + lane;
                item[k] = make_int2(-1, i);
                if (i < hi) {
                    if (p == 0) item[k].x = valid_row(load_id(s.ids, s.id64, i), s.V, status);
                    else item[k] = __ldcg(in + i);
                }
            }
        };
        for (int i = lane; i < bins; i += 32) mine[i] = 0;
        __syncwarp();
        int2 item[kSortKeys];
        for (int i0 = lo; i0 < hi; i0 += 32 * kSortKeys) {
            load(i0, item, s.status);
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
                if (item[k].x >= 0) atomicAdd(&mine[(item[k].x >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        if (tid < bins) {
            int sum = 0;
#pragma unroll 8
            for (int w = 0; w < kClusterWarps; ++w) {
                const int c = sh[w * kMaxBins + tid];
                sh[w * kMaxBins + tid] = sum;
                sum += c;
            }
            total[tid] = sum;
        }
        cluster.sync();
        int all = 0, before = 0;
        if (tid < bins) {
#pragma unroll
            for (int r = 0; r < kClusterBlocks; ++r) {
                const int c = cluster.map_shared_rank(total, r)[tid];
                all += c;
                if (r < rank) before += c;
            }
        }
        int incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        int base = incl - all;
        n = 0;  // from the first pass on, the valid ids
#pragma unroll
        for (int w = 0; w < kMaxBins / 32; ++w) {
            const int c = scan[w];
            if (w < warp) base += c;
            n += c;
        }
        if (tid < bins) offset[tid] = base + before;
        __syncthreads();
        const bool once = lo + 32 * kSortKeys >= hi;  // the keys are still in registers
        for (int i0 = lo; i0 < hi; i0 += 32 * kSortKeys) {
            if (!once) load(i0, item, nullptr);
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k) {
                if (i0 + k * 32 >= hi) break;
                const int digit = (item[k].x >> shift) & (bins - 1);
                unsigned same = __ballot_sync(0xffffffffu, item[k].x >= 0);  // lanes with this lane's digit
                for (int b = 0; b < s.bits; ++b) {
                    const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1);
                    same &= ((digit >> b) & 1) ? set : ~set;
                }
                const unsigned lower = same & ((1u << lane) - 1);
                int prior = 0;
                if (item[k].x >= 0) prior = mine[digit];
                __syncwarp();
                if (item[k].x >= 0 && lower == 0) mine[digit] = prior + __popc(same);
                __syncwarp();
                if (item[k].x >= 0) out[offset[digit] + prior + __popc(lower)] = item[k];
            }
        }
        cluster.sync();
    }
    if (rank == 0 && tid == 0) *s.n_valid = n;
}

// ---- gradient: sums of the sorted runs

constexpr int kPiece = 32;

struct RunArgs {
    const int2* items;   // (key, position), sorted, in whole pieces
    const int32_t* n_valid;
    float* part;         // [pieces][2][ld_part]: a run from the piece before, a run into the next
    int64_t ld_part;
    int64_t ld, ld_out;
    int64_t count;       // ids, valid or not
    int cols;            // wide columns (D / VEC)
    int spans;           // ceil(cols / 32)
    float scale;
    int accumulate;
};

// *p += f without waiting for what was there. Each element is added to once in a call, so that no order of
// the adds can change it.
template <int N>
__device__ __forceinline__ void add_at(float* p, const float* f) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + i), "f"(f[i]), "f"(f[i + 1]), "f"(f[i + 2]), "f"(f[i + 3]) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p + i), "f"(f[i]) : "memory");
    }
}

template <class O, int VEC>
__device__ __forceinline__ void finish_row(const RunArgs& a, O* out, int32_t key, int v, float* acc) {
    O* o = out + (int64_t)key * a.ld_out + (int64_t)v * VEC;
    if (sizeof(O) == 2 && a.accumulate) {
        float old[VEC];
        load_n<O, VEC>(o, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(acc[i], a.scale, old[i]);
        store_n<O, VEC>(o, acc);
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
    if constexpr (sizeof(O) == 4) {
        if (a.accumulate) return add_at<VEC>(o, acc);
    }
    store_n<O, VEC>(o, acc);
}

// LANES lanes sum one piece over one span of columns. BATCH rows are loaded together, and where a 16-bit table
// is added to (ACC), what it holds at the runs that end among them. It is bound by how many loads of rows are in
// flight: for wide rows four a lane and 32 warps an SM (28,800 x 960 bf16 rows: the gradient takes 47 us, with
// eight and 20 warps 52 us), for narrow ones, whose warps hold two or four pieces, eight (256,000 x 128 bf16: 63
// and with four 65 us).
template <class T, class O, int VEC, int LANES, bool ACC>
__global__ void __launch_bounds__(256, LANES == 32 && !(ACC && sizeof(O) == 2) ? 4 : 2) run_sum_kernel(RunArgs a, const T* __restrict__ grad, O* __restrict__ out) {
    constexpr int BATCH = LANES == 32 ? 4 : 8;
    wait_for_previous();
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int64_t piece = unit / a.spans;
    const int v = (int)(unit - piece * a.spans) * LANES + lane;
    const int n = *a.n_valid;
    const int64_t first = piece * kPiece;
    if (first >= n || v >= a.cols) return;
    const int m = (int)min((int64_t)kPiece, n - first);
    const int32_t prev = first > 0 ? a.items[first - 1].x : -1;
    const int32_t next = first + m < n ? a.items[first + m].x : -1;
    const T* col = grad + (int64_t)v * VEC;
    float acc[VEC] = {};
    bool from_before = false;
    auto to_slot = [&](int which) { store_n<float, VEC>(a.part + (piece * 2 + which) * a.ld_part + (int64_t)v * VEC, acc); };
    for (int j0 = 0; j0 < m; j0 += BATCH) {
        int32_t key[BATCH + 1], pos[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k += 2) {
            const int4 two = *reinterpret_cast<const int4*>(a.items + first + j0 + k);
            key[k] = two.x;
            pos[k] = two.y;
            key[k + 1] = two.z;
            pos[k + 1] = two.w;
        }
        key[BATCH] = j0 + BATCH < m ? a.items[first + j0 + BATCH].x : next;
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            if (j0 + k >= m) key[k] = next;  // -1 there: past the last id
        Pack<T, VEC> p[BATCH];
        constexpr bool OLD = ACC && sizeof(O) == 2;
        Pack<O, sizeof(O) == 2 ? VEC : 1> old[OLD ? BATCH : 1];
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            if (j0 + k < m) p[k] = Pack<T, VEC>::load_stream(col + (int64_t)pos[k] * a.ld);
        if constexpr (OLD) {
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
                if (j0 + k < m && key[k + 1] != key[k]) old[k] = Pack<O, VEC>::load(out + (int64_t)key[k] * a.ld_out + (int64_t)v * VEC);
        }
        if (j0 == 0) from_before = prev == key[0];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            if (j0 + k >= m) break;
            float f[VEC];
            p[k].get(f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += f[i];
            if (key[k + 1] != key[k]) {  // the run's end
                if (from_before) {
                    to_slot(0);
                    from_before = false;
                } else {
                    O* o = out + (int64_t)key[k] * a.ld_out + (int64_t)v * VEC;
                    if constexpr (OLD) {
                        float was[VEC];
                        old[k].get(was);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(acc[i], a.scale, was[i]);
                        store_n<O, VEC>(o, acc);
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
                        if constexpr (ACC) add_at<VEC>(o, acc);
                        else store_n<O, VEC>(o, acc);
                    }
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
            }
        }
    }
    if (m == kPiece && next == a.items[first + kPiece - 1].x) to_slot(from_before ? 0 : 1);  // into the next piece
}

constexpr int kJoinAlone = 16;  // partial sums that one warp adds by itself

// Adds the partial sums of each run that crosses pieces: slot 1 of its first piece, then slot 0 of the
// others. One warp per (piece, span of LANES wide columns); its 32 / LANES sets of lanes take turns of the
// partial sums, and a long run is shared by the block's 8 warps.
template <class O, int VEC, int LANES>
__global__ void __launch_bounds__(256) run_join_kernel(RunArgs a, O* __restrict__ out) {
    __shared__ int64_t long_first[8], long_last[8];
    __shared__ int32_t long_key[8];
    __shared__ __align__(16) float sums[8][LANES * VEC];
    constexpr int SETS = 32 / LANES;
    wait_for_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, set = lane / LANES;
    const int64_t group = blockIdx.x / a.spans;
    const int v = (int)(blockIdx.x % a.spans) * LANES + (lane & (LANES - 1));
    const bool on = v < a.cols;
    const int64_t piece = group * 8 + warp;
    // the sum of slot 0 of pieces [lo, hi), and of slot 1 of piece `head` if it is one (>= 0), in every lane
    auto add = [&](float* acc, int64_t head, int64_t lo, int64_t hi) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        if (on) {
            if (head >= 0 && set == 0) load_n<float, VEC>(a.part + (head * 2 + 1) * a.ld_part + (int64_t)v * VEC, acc);
#pragma unroll 8
            for (int64_t q = lo + (head >= 0 ? (set + SETS - 1) % SETS : set); q < hi; q += SETS) {
                float f[VEC];
                load_n<float, VEC>(a.part + q * 2 * a.ld_part + (int64_t)v * VEC, f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += f[i];
            }
        }
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
        }
    };
    bool is_long = false;
    const int64_t end = (piece + 1) * kPiece;
    if (end < a.count) {
        // everything that the first decisions need, at once (n bounds what of it is meant)
        const int n = *a.n_valid;
        const int32_t key = a.items[end - 1].x, after = a.items[end].x, head = a.items[end - kPiece].x;
        const int32_t before = piece > 0 ? a.items[end - kPiece - 1].x : -1;
        // piece q's first key, and whether the run of `key` reaches its end
        auto probe = [&](int64_t q, int32_t& first_key) {
            first_key = q * kPiece < a.count ? a.items[q * kPiece].x : -1;
            return (q + 1) * kPiece <= n && a.items[(q + 1) * kPiece - 1].x == key;
        };
        int32_t first_key;
        int64_t known = piece;  // the run reaches this piece's end
        unsigned miss = ~__ballot_sync(0xffffffffu, probe(known + 1 + lane, first_key));
        if (end < n && after == key && (head != key || before != key)) {
            if (miss == 0) {  // in steps of 32 pieces, then the last 32
                known += 32;
                while ((miss = ~__ballot_sync(0xffffffffu, probe(known + 32 * (lane + 1), first_key))) == 0) known += 1024;
                known += 32 * (__ffs(miss) - 1);
                miss = ~__ballot_sync(0xffffffffu, probe(known + 1 + lane, first_key));
            }
            int64_t last = known + __ffs(miss);
            if (last * kPiece >= n || __shfl_sync(0xffffffffu, first_key, __ffs(miss) - 1) != key) --last;  // ended before
            if (last - piece < kJoinAlone) {
                float acc[VEC];
                add(acc, piece, piece + 1, last + 1);
                if (on && set == 0) finish_row<O, VEC>(a, out, key, v, acc);
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
        float acc[VEC];
        add(acc, warp == 0 ? long_first[r] : -1, lo + m * warp / 8, lo + m * (warp + 1) / 8);
        if (set == 0) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sums[warp][lane * VEC + i] = acc[i];
        }
        __syncthreads();
        if (warp == 0 && set == 0 && on) {
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
    int2* items[2];
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
    if (T > kDirectIds) {
        w.n_valid = (int32_t*)take(256);
        const size_t pieces = (size_t)((T + kPiece - 1) / kPiece);
        w.counts = (int32_t*)take((size_t)kMaxTiles * kMaxBins * 4);
        for (int i = 0; i < 2; ++i) w.items[i] = (int2*)take(pieces * kPiece * sizeof(int2));
        w.part = (float*)take(pieces * 2 * part_stride(D) * 4);
    }
    if (ws) *ws = w;
    return off;
}

cudaLaunchConfig_t cluster_config(cudaLaunchAttribute* attr, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kClusterBlocks);
    cfg.blockDim = dim3(kClusterThreads);
    cfg.dynamicSmemBytes = kClusterSmem;
    cfg.stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = kClusterBlocks;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

// Whether the current device has room for the cluster (it needs kClusterBlocks SMs that share a GPC); asked once.
bool cluster_fits() {
    static std::atomic<int> known[64];  // 0: not asked, 1: no, 2: yes
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int k = known[dev].load(std::memory_order_relaxed);
    if (k == 0) {
        cudaLaunchAttribute attr;
        const cudaLaunchConfig_t cfg = cluster_config(&attr, nullptr);
        int n = 0;
        const bool ok = cudaFuncSetAttribute(sort_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                        allow_smem<sort_cluster_kernel>(kClusterSmem) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&n, sort_cluster_kernel, &cfg) == cudaSuccess && n > 0;
        if (!ok) cudaGetLastError();
        k = ok ? 2 : 1;
        known[dev].store(k, std::memory_order_relaxed);
    }
    return k == 2;
}

// Zeros that take longer than a fork and a join of streams cost are written beside the sort: 8 MB, 31 us for 16,000
// ids in place of 33 us; 61 MB, 35 in place of 45 us.
constexpr int64_t kSideZeros = 4 << 20;

// Work on the side stream that the caller's stream has to wait for, whichever way the call ends.
struct Beside {
    SideStream* ss;
    cudaStream_t st;
    cudaError_t join() {
        if (!ss) return cudaSuccess;
        SideStream* s = ss;
        ss = nullptr;
        const cudaError_t e = cudaEventRecord(s->join, s->s);
        return e != cudaSuccess ? e : cudaStreamWaitEvent(st, s->join, 0);
    }
    ~Beside() { join(); }
};

template <class T, class O>
cudaError_t grad_typed(const T* grad, int64_t ld, const void* ids, int id64, int64_t count, int64_t V, int D, float scale,
                       int accumulate, O* out, int64_t ld_out, void* workspace, int32_t* status, int* launches,
                       cudaStream_t st) {
    cudaError_t e;
    constexpr int kMax = 16 / (int)sizeof(T);
    int vec = wide_elements({{grad, ld, (int)sizeof(T)}, {out, ld_out, (int)sizeof(O)}}, D, kMax);
    Beside side{nullptr, st};  // zeros are written beside the sort
    if (!accumulate && V > 0) {
        const int64_t row_bytes = (int64_t)D * sizeof(O);
        cudaStream_t zs = st;
        if (count > kDirectIds && V * row_bytes >= kSideZeros) {
            SideStream* ss = nullptr;
            if ((e = side_stream(&ss)) != cudaSuccess) return e;
            if ((e = cudaEventRecord(ss->fork, st)) != cudaSuccess) return e;
            if ((e = cudaStreamWaitEvent(ss->s, ss->fork, 0)) != cudaSuccess) return e;
            side.ss = ss;
            zs = ss->s;
        }
        e = ld_out == D ? cudaMemsetAsync(out, 0, (size_t)V * row_bytes, zs)
                        : cudaMemset2DAsync(out, ld_out * sizeof(O), 0, (size_t)row_bytes, V, zs);
        if (e != cudaSuccess) return e;
    }
    if (count == 0) return cudaSuccess;
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
    const int passes = (bits + 8) / 9, pass_bits = (bits + passes - 1) / passes;
    if (count <= kClusterIds && cluster_fits()) {
        ClusterSort s;
        s.ids = ids;
        s.id64 = id64;
        s.V = V;
        s.count = (int)count;
        s.bits = pass_bits;
        s.passes = passes;
        for (int i = 0; i < 2; ++i) s.items[i] = ws.items[i];
        s.n_valid = ws.n_valid;
        s.status = status;
        cudaLaunchAttribute attr;
        const cudaLaunchConfig_t cfg = cluster_config(&attr, st);
        if ((e = cudaLaunchKernelEx(&cfg, sort_cluster_kernel, s)) != cudaSuccess) return e;
        *launches += 1;
    } else {
        SortPass s;
        s.ids = ids;
        s.id64 = id64;
        s.V = V;
        s.n_valid = ws.n_valid;
        s.count = count;
        s.bits = pass_bits;
        s.tile = ((count + kMaxTiles - 1) / kMaxTiles + kSubTile - 1) / kSubTile * kSubTile;
        const int tiles = (int)((count + s.tile - 1) / s.tile);
        constexpr int kSmem = kSortWarps * kMaxBins * 4 + kSubTile * (int)sizeof(int2);
        if ((e = allow_smem<sort_scatter_kernel>(kSmem)) != cudaSuccess) return e;
        for (int p = 0; p < passes; ++p) {
            s.first = p == 0;
            s.shift = p * s.bits;
            s.in = ws.items[(p + 1) & 1];
            s.out = ws.items[p & 1];
            if (p == 0) sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(s, ws.counts, status);
            else if ((e = launch_chained(sort_count_kernel, tiles, kSortThreads, 0, st, s, ws.counts, status)) != cudaSuccess) return e;
            if ((e = launch_chained(sort_scatter_kernel, tiles, kSortThreads, kSmem, st, s, ws.counts, tiles)) != cudaSuccess) return e;
        }
        *launches += 2 * passes;
    }
    const bool joined = side.ss != nullptr;
    if ((e = side.join()) != cudaSuccess) return e;
    RunArgs a;
    a.items = ws.items[(passes - 1) & 1];
    a.count = count;
    a.n_valid = ws.n_valid;
    a.part = ws.part;
    a.ld_part = part_stride(D);
    a.ld = ld;
    a.ld_out = ld_out;
    a.scale = scale;
    a.accumulate = accumulate;
    a.cols = D / vec;
    const int64_t pieces = (count + kPiece - 1) / kPiece;
    const int lanes = a.cols > 16 ? 32 : a.cols > 8 ? 16 : 8;
    a.spans = (a.cols + lanes - 1) / lanes;
    const int64_t grid = (pieces * a.spans * lanes + 255) / 256, join_grid = (pieces + 7) / 8 * a.spans;
    if (grid > 0x7fffffff || join_grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    with_vec<kMax>(vec, [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        auto go = [&](auto l) {
            constexpr int LANES = decltype(l)::value;
            const auto sum = accumulate ? run_sum_kernel<T, O, VEC, LANES, true> : run_sum_kernel<T, O, VEC, LANES, false>;
            if (joined) {
                sum<<<(unsigned)grid, 256, 0, st>>>(a, grad, out);
                e = cudaGetLastError();
            } else {
                e = launch_chained(sum, grid, 256, 0, st, a, grad, out);
            }
            if (e == cudaSuccess) e = launch_chained(run_join_kernel<O, VEC, LANES>, join_grid, 256, 0, st, a, out);
        };
        if (lanes == 32) go(std::integral_constant<int, 32>{});
        else if (lanes == 16) go(std::integral_constant<int, 16>{});
        else go(std::integral_constant<int, 8>{});
    });
    *launches += 2;
    return e;
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
