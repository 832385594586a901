// Kernels of the paged KV cache held in 4 bits (host side: kv4.cu; entry points: include/vuib200.h, "Paged KV cache in 4 bits").
//
// A stored vector (one position, one kv head, keys or values) is cut into groups of 32 elements:
//   zero = f16(min x), scale = f16((max x - zero) * fl(1/15)), code = rint((x - zero) / scale) in 0 .. 15,
// and a code stands for f16(scale * code + zero).  (Attention of up to 4 columns takes scale * code + zero as it is.)
//
// Layout of a layer's pool: [block][kv head][16 positions][32 elements] -> 640 bytes, laid out as the fragments that the attention
// feeds to the tensor cores (lane = 4 g + t of a warp; keys 0 .. 15 are the positions of a tile):
//   [  0, 256)  key codes: lane's 8 bytes = word of key g, word of key g + 8; nibble j of a word's low half is element 8 t + 2 j,
//               of its high half element 8 t + 2 j + 1
//   [256, 320)  key scale and zero: (scale, zero) of key g, of key g + 8, g = 0 .. 7
//   [320, 576)  value codes: lane's 8 bytes = two words, each a byte of the keys 2t, 2t+8, 2t+1, 2t+9; a byte of the first word holds
//               elements 4 g (low nibble) and 4 g + 1, of the second 4 g + 2 and 4 g + 3
//   [576, 640)  value scale and zero, as the keys'
// So a tile is read with one 8-byte load a lane and operand, without a shuffle, and a position owns whole words (keys) and bytes
// (values): storing one position never reads or rewrites another's.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vuik {

constexpr int KV4_GROUP = 32;
constexpr int KV4_TILE = 16;              // positions of a tile
constexpr int KV4_GT = 640;               // bytes of a tile's group
constexpr int KV4_KPAR = 256, KV4_VCODE = 320, KV4_VPAR = 576;
static_assert(KV4_VCODE == KV4_GT / 2 && KV4_VPAR - KV4_VCODE == KV4_KPAR, "a group's values lie as its keys do");
constexpr float KV4_LIMIT = 60000.f;      // larger magnitudes are stored as this (f16 ends at 65504)
constexpr int KV4_MAX_SEQS = 4096;

// bits of the device flag
constexpr int KV4_BAD_SLOT = 1, KV4_BAD_LEN = 2, KV4_NO_ROWS = 4, KV4_NO_BLOCKS = 8, KV4_BAD_VALUE = 16, KV4_BAD_BLOCK = 32, KV4_TIMEOUT = 64;
constexpr unsigned KV4_POLLS = 1u << 22;  // bound of every wait

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// What all kernels know of a cache.  (A plan's entry is an int4: slot, -1 if it takes no part; first new position; rows; first row.)
struct Kv4Cache {
    unsigned char* pool;        // of the layer
    int32_t* table;             // (max_seqs, max_blocks)
    int32_t* lens;
    int32_t* free_blocks;
    int32_t* n_free;
    int32_t* flag;
    int n_kv, block_shift, n_blocks, max_seqs, max_blocks;
};

// Positions of a split of attention's work: by the length of the sequence alone, so that a row's bits do not depend on what else is there.
struct Kv4Split {
    int up_to_512, up_to_1024, beyond;
    int most;        // splits of one sequence: longer ones get larger splits, multiples of 256 positions, so that a stage ends with its split
    bool weigh;      // units count for what they cost: their positions by 64, and one more
    __host__ __device__ int of(long long len) const {
        const int s = len <= 512 ? up_to_512 : len <= 1024 ? up_to_1024 : beyond;
        return (long long)s * most >= len ? s : (int)(((len + most - 1) / most + 255) & ~255ll);
    }
    __host__ __device__ int parts(long long len) const { const int s = of(len); return (int)((len + s - 1) / s); }
    __host__ __device__ int work(long long len) const { return parts(len) + (weigh ? (int)((len + 63) / 64) : 0); }     // of all parts
    __host__ __device__ int work_of(int positions) const { return 1 + (weigh ? (positions + 63) / 64 : 0); }            // of one
};

// ------------------------------------------------------------------------------------------------ tables and maps
struct Kv4PlanArgs {
    Kv4Cache c;
    const int32_t* slots; const int32_t* new_lens; const int32_t* at;
    int n, n_rows, max_new;
    int group, cols;            // query heads a kv head, columns of a tile: attention's units are counted here
    Kv4Split split;
    int4* entries; int32_t* cu_units; int32_t* cu_work; int32_t* cu_tiles; int32_t* row_entry;    // the plan's work array
    int32_t* cu_rows; int32_t* row_slot; int32_t* row_pos; long long* slot_map;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned cluster_size() { unsigned r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }

// What the CTAs of the cluster (or the one CTA) wrote to global memory before is seen by all of them behind it, when read from the L2.
__device__ __forceinline__ void plan_sync(unsigned size) {
    if (size == 1) { __syncthreads(); return; }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive prefix sums over the block of N non-negative numbers a thread, side by side; v becomes the sum before the thread, total the
// whole.  Sums stop at KV4_MANY, which no size that can be served reaches; two of them still fit an int.
constexpr int KV4_MANY = (1 << 30) - 1;
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (*warp_sums)[32], int (&total)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = v[j];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int y = __shfl_up_sync(0xffffffffu, x[j], o);
            if (lane >= o) x[j] = min(x[j] + y, KV4_MANY);
        }
    }
    if (lane == 31) {
#pragma unroll
        for (int j = 0; j < N; ++j) warp_sums[j][warp] = x[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int s = lane < nw ? warp_sums[j][lane] : 0;
        int p = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) p = min(p + y, KV4_MANY);
        }
        total[j] = __shfl_sync(0xffffffffu, p, 31);
        const int excl = __shfl_up_sync(0xffffffffu, p, 1);
        const int before = __shfl_sync(0xffffffffu, lane ? excl : 0, warp);
        const int in = __shfl_up_sync(0xffffffffu, x[j], 1);
        v[j] = min(before + (lane ? in : 0), KV4_MANY);
    }
}

// The last i with first[i] <= x, for a non-decreasing first[0 .. n] with first[0] = 0 and x < first[n].
__device__ __forceinline__ int find_in(const int* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// One CTA, or one cluster whose CTAs all compute the same few prefix sums and share out what is written: a step's entries are few, its
// rows and blocks many.  Latency bound: three dependent reads (entry, length, table) and five barriers.  64 sequences of one row: 5.6 us a call in a
// graph; 512 sequences emptied, then filled again with 4 to 300 positions each (81000 rows): 15 us each of the two calls.
__global__ void __launch_bounds__(1024) k_kv4_plan(const Kv4PlanArgs a) {
    extern __shared__ int sm[];
    __shared__ int scan_a[1][32], scan_b[2][32], scan_c[5][32];
    const int n = a.n, per = (n + blockDim.x - 1) / blockDim.x;
    int* s_slot = sm;               // n each; slot -1: takes no part
    int* s_start = s_slot + n;
    int* s_new = s_start + n;
    int* s_have = s_new + n;
    int* s_need = s_have + n;
    int* s_cu = s_need + n;         // n + 1 each
    int* s_grow = s_cu + n + 1;
    int* s_drop = s_grow + n + 1;
    int* owner = s_drop + n + 1;    // max_seqs
    const unsigned size = cluster_size(), rank = cluster_rank();
    const int tid = threadIdx.x, first = tid * per, last = min(n, first + per);
    const int bs = 1 << a.c.block_shift;
    const long long max_len = (long long)a.c.max_blocks << a.c.block_shift;
    int bad = 0;

    for (int i = tid; i < a.c.max_seqs; i += blockDim.x) owner[i] = n;
    pdl_wait();
    pdl_launch();
    const int n_free = __ldcg(a.c.n_free);
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        const int slot = __ldcg(a.slots + i);
        s_slot[i] = slot;
        if (slot >= 0 && slot < a.c.max_seqs) atomicMin(owner + slot, i);
    }
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        int slot = s_slot[i];
        const bool there = slot >= 0 && slot < a.c.max_seqs && owner[slot] == i;   // a slot's first entry counts
        if (!there && slot != -1) bad |= KV4_BAD_SLOT;
        int len = 0, start = 0;
        long long want = 0;
        bool ok = there;
        if (there) {
            len = __ldcg(a.c.lens + slot);
            want = a.new_lens ? __ldcg(a.new_lens + i) : 1;
            start = a.at ? __ldcg(a.at + i) : len;
            if (len < 0 || len > max_len || start < 0 || start > len || want < 0 || want > a.max_new || start + want > max_len) {
                bad |= KV4_BAD_LEN;
                ok = false;
            }
        }
        s_slot[i] = ok ? slot : -1;
        s_start[i] = ok ? start : 0;
        s_new[i] = ok ? (int)want : 0;
        s_have[i] = ok ? (len + bs - 1) >> a.c.block_shift : 0;
        s_need[i] = ok ? (int)((start + want + bs - 1) >> a.c.block_shift) : 0;
    }
    __syncthreads();
    // Who is served: the rows of the entries so far have to fit, and so have the blocks that they ask for (an entry that asks for none
    // is served all the same).
    auto leave_out = [&](int i) { s_slot[i] = -1; s_new[i] = 0; s_need[i] = s_have[i]; };
    int rows_to[1] = {0}, all[1];
    for (int i = first; i < last; ++i) rows_to[0] = min(rows_to[0] + s_new[i], KV4_MANY);
    block_scan<1>(rows_to, scan_a, all);
    int blocks[2] = {0, 0}, sum[2];     // given back, asked for
    for (int i = first; i < last; ++i) {
        rows_to[0] = min(rows_to[0] + s_new[i], KV4_MANY);
        if (rows_to[0] > a.n_rows) {
            if (s_slot[i] >= 0) bad |= KV4_NO_ROWS;
            leave_out(i);
        }
        blocks[0] += max(s_have[i] - s_need[i], 0);
        blocks[1] = min(blocks[1] + max(s_need[i] - s_have[i], 0), KV4_MANY);
    }
    block_scan<2>(blocks, scan_b, sum);
    const int dropped = sum[0], top = n_free + dropped;
    int part[5] = {0, 0, 0, 0, 0}, whole[5];   // blocks got, rows, units of attention (of a kv head) and their work, tiles of 16 positions written
    auto times_tiles = [&](int i, int of_one) { return (int)min(((long long)s_new[i] * a.group + a.cols - 1) / a.cols * of_one, (long long)KV4_MANY); };
    auto units_of = [&](int i) { return s_new[i] ? times_tiles(i, a.split.parts(s_start[i] + (long long)s_new[i])) : 0; };
    auto work_of = [&](int i) { return s_new[i] ? times_tiles(i, a.split.work(s_start[i] + (long long)s_new[i])) : 0; };
    auto tiles_of = [&](int i) { return s_new[i] ? ((s_start[i] + s_new[i] - 1) >> 4) - (s_start[i] >> 4) + 1 : 0; };
    for (int i = first; i < last; ++i) {
        s_drop[i] = blocks[0];
        blocks[0] += max(s_have[i] - s_need[i], 0);
        const int g = max(s_need[i] - s_have[i], 0);
        blocks[1] = min(blocks[1] + g, KV4_MANY);
        if (g > 0 && blocks[1] > top) {
            bad |= KV4_NO_BLOCKS;
            leave_out(i);
        } else {
            part[0] += g;
        }
        part[1] += s_new[i];
        part[2] = min(part[2] + units_of(i), KV4_MANY);
        part[3] = min(part[3] + work_of(i), KV4_MANY);
        part[4] += tiles_of(i);
    }
    block_scan<5>(part, scan_c, whole);
    const int grown = whole[0], rows = whole[1];
    int units = part[2], work = part[3], tiles = part[4];
    for (int i = first; i < last; ++i) {
        s_grow[i] = part[0];
        s_cu[i] = part[1];
        part[0] += max(s_need[i] - s_have[i], 0);
        part[1] += s_new[i];
    }
    if (tid == 0) { s_cu[n] = rows; s_grow[n] = grown; s_drop[n] = dropped; }
    if (bad && rank == 0) atomicOr(a.c.flag, bad);
    __syncwarp();
    plan_sync(size);                   // every CTA has read the lengths and the number of free blocks
    const int step = blockDim.x * size, me = rank * blockDim.x + tid;
    if (rank == 0) {
        if (tid == 0) {
            *a.c.n_free = top - grown;
            a.cu_rows[n] = rows;
            a.cu_units[n] = whole[2];
            a.cu_work[n] = whole[3];
            a.cu_tiles[n] = whole[4];
        }
        for (int i = first; i < last; ++i) {
            a.cu_units[i] = units;
            a.cu_work[i] = work;
            a.cu_tiles[i] = tiles;
            units = min(units + units_of(i), KV4_MANY);
            work = min(work + work_of(i), KV4_MANY);
            tiles += tiles_of(i);
            a.cu_rows[i] = s_cu[i];
            a.entries[i] = make_int4(s_slot[i], s_start[i], s_new[i], s_cu[i]);
            if (s_slot[i] >= 0) a.c.lens[s_slot[i]] = s_start[i] + s_new[i];
        }
    }
    // Blocks given back go on the stack so that the first entry's first one is on top; those taken come off the top in entry order:
    // what was given back and is taken again in the same order gets its places again.
    // Four at a time, so that their reads of the L2 are under way together.
    for (int r0 = me; r0 < dropped; r0 += 4 * step) {
        int32_t* at[4];
        int id[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + k * step;
            at[k] = nullptr;
            if (r >= dropped) continue;
            const int i = find_in(s_drop, n, r);
            at[k] = a.c.table + (size_t)s_slot[i] * a.c.max_blocks + s_need[i] + (r - s_drop[i]);
            id[k] = __ldcg(at[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!at[k]) continue;
            const int to = top - 1 - (r0 + k * step);
            if (to < a.c.n_blocks) a.c.free_blocks[to] = id[k];
            *at[k] = -1;
        }
    }
    if (dropped) plan_sync(size);
    for (int r0 = me; r0 < grown; r0 += 4 * step) {
        int32_t* at[4];
        int id[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + k * step;
            at[k] = nullptr;
            if (r >= grown) continue;
            id[k] = __ldcg(a.c.free_blocks + (top - 1 - r));
            const int i = find_in(s_grow, n, r);
            at[k] = a.c.table + (size_t)s_slot[i] * a.c.max_blocks + s_have[i] + (r - s_grow[i]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at[k]) *at[k] = id[k];
    }
    if (grown || dropped) plan_sync(size);
    for (int r0 = me; r0 < a.n_rows; r0 += 4 * step) {
        int entry[4], pos[4], block[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + k * step;
            entry[k] = pos[k] = block[k] = -1;
            if (r >= rows) continue;
            const int i = find_in(s_cu, n, r);
            entry[k] = i;
            pos[k] = s_start[i] + (r - s_cu[i]);
            block[k] = __ldcg(a.c.table + (size_t)s_slot[i] * a.c.max_blocks + (pos[k] >> a.c.block_shift));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + k * step;
            if (r >= a.n_rows) continue;
            const bool fine = (unsigned)block[k] < (unsigned)a.c.n_blocks;
            if (!fine && entry[k] >= 0) atomicOr(a.c.flag, KV4_BAD_BLOCK);
            a.row_entry[r] = entry[k];
            a.row_slot[r] = entry[k] >= 0 ? s_slot[entry[k]] : -1;
            a.row_pos[r] = pos[k];
            a.slot_map[r] = fine ? ((long long)block[k] << a.c.block_shift) + (pos[k] & (bs - 1)) : -1;
        }
    }
}

__global__ void k_kv4_reset(Kv4Cache c) {
    const long long n = (long long)c.max_seqs * c.max_blocks, step = (long long)gridDim.x * blockDim.x;
    const long long me = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    pdl_wait();
    for (long long i = me; i < n; i += step) c.table[i] = -1;
    for (long long i = me; i < c.n_blocks; i += step) c.free_blocks[i] = (int)i;
    for (long long i = me; i < c.max_seqs; i += step) c.lens[i] = 0;
    if (me == 0) { *c.n_free = c.n_blocks; *c.flag = 0; }
}

// ------------------------------------------------------------------------------------------------ rows in and out
// Byte offset of the tile of position `where` (block * block size + offset in it), kv head h, in a layer's pool.
template <int NG>
__device__ __forceinline__ size_t tile_at(const Kv4Cache& c, long long where, int h) {
    const int tiles = 1 << (c.block_shift - 4);
    const long long b = where >> c.block_shift;
    const int tile = (int)(where & ((1 << c.block_shift) - 1)) >> 4;
    return ((size_t)(b * c.n_kv + h) * tiles + tile) * (NG * KV4_GT);
}

struct Kv4RowsArgs {
    Kv4Cache c;
    const __nv_bfloat16* k; const __nv_bfloat16* v;      // append: rows in
    __nv_bfloat16* k_out; __nv_bfloat16* v_out;          // read: rows out
    long long k_stride, v_stride;                        // elements between rows
    const int4* entries; const int32_t* cu_tiles; int n; // append: the plan's entries, their first tiles
    const int32_t* row_slot; const int32_t* row_pos;     // read
    int n_rows;
};

// The largest magnitude of 8 bf16 as bits (infinity and NaN are larger than any number).
__device__ __forceinline__ uint32_t most_bits(const uint4& r) {
    const uint32_t m = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}

__device__ __forceinline__ float tame(float x) { return x == x ? fminf(fmaxf(x, -KV4_LIMIT), KV4_LIMIT) : 0.f; }
// Element j of 16 bf16.
__device__ __forceinline__ float element(const uint32_t (&w)[8], int j) { return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }

// Which of the codes k and k + 1 (k = 0 .. 14) the quotient f / s, rounded to fp32, rounds to; it is within 2^-16 of their middle t.  The distance
// f - t s is exact (t s has 15 bits, f is next to it); the quotient rounds to t itself, and then to the even code, if it is half a unit in
// the last place of t off or less (below 0.5, a power of two, units are half as large).
__device__ __forceinline__ float code_between(float f, float s, float k) {
    const float t = k + 0.5f, r = fmaf(-t, s, f), half_ulp = __int_as_float((__float_as_int(t) & 0x7f800000) - (24 << 23)) * s;
    const bool up = r > half_ulp, down = r < (k == 0.f ? -0.5f * half_ulp : -half_ulp);
    return k + (up || (!down && ((int)k & 1)) ? 1.f : 0.f);
}

// A warp stores the keys or the values (blockIdx.y) of one tile of 16 positions of one kv head, or of those of its positions that are new: 16
// elements a lane, two lanes a group, which share its extremes; the codes are gathered in shared memory as they lie in the pool and leave
// it 16 bytes a lane where the whole tile is new, else in the words and bytes of the new positions.
// The nearest code: (x - zero) times the reciprocal of 15 scales, kept within [0, 1] and times 15, is 2^-17.4 off at most (a division of two ulp and two roundings, of a
// quotient below 16), so unless that lies within 2^-17 of the middle between two codes it rounds as the quotient does; lanes that have such an
// element (exact middles are not rare among bf16 numbers: one group of normal ones in fifty) look closer.
// Bound by instructions: 16000 rows of 8 heads of 128 are 33 million elements, 22 an element and lane; 37 us (65 MB in and 20 out: 13 us).  Keys and
// values in one warp, unrolled, took 72 us (50 KB of code), 8 elements a lane with a division each 55.
template <int NG>
__global__ void __launch_bounds__(128) k_kv4_append(const Kv4RowsArgs a) {
    constexpr int LANES = NG * 2, ROWS = 32 / LANES;     // lanes of a row; rows side by side: 8, 5 (2 lanes idle), 4
    constexpr float NEAR = 0.5f - 7.62939453125e-6f;         // 2^-17 from the middle between two codes
    constexpr int PITCH = KV4_GT / 2 + 16;                       // a group's image: 4 banks further than the one before
    __shared__ __align__(16) unsigned char image[4][NG * PITCH];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* const img = image[warp];
    const long long id = (long long)blockIdx.x * 4 + warp;
    const int h = (int)(id % a.c.n_kv), want = (int)(id / a.c.n_kv);
    const bool half = blockIdx.y != 0;         // values
    pdl_wait();
    pdl_launch();
    int lo = 0, hi = a.n;      // the entry that tile number `want` belongs to
    if (want >= __ldcg(a.cu_tiles + a.n)) return;
    int before = 0;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const int f = at < hi ? __ldcg(a.cu_tiles + at) : 0x7fffffff;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, f <= want));
        before = __shfl_sync(0xffffffffu, f, k);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    const int4 e = __ldcg(a.entries + lo);
    const int pos0 = ((e.y >> 4) + want - before) << 4;                       // the tile's first position
    const int from = max(e.y, pos0) - pos0, to = min(e.y + e.z, pos0 + 16) - pos0;
    const int b = __ldcg(a.c.table + (size_t)e.x * a.c.max_blocks + (pos0 >> a.c.block_shift));
    if ((unsigned)b >= (unsigned)a.c.n_blocks) {
        if (lane == 0) atomicOr(a.c.flag, KV4_BAD_BLOCK);
        return;
    }
    unsigned char* const tile = a.c.pool + tile_at<NG>(a.c, ((long long)b << a.c.block_shift) + (pos0 & ((1 << a.c.block_shift) - 1)), h);
    const int sub = lane / LANES, ch = lane % LANES;
    unsigned char* const gimg = img + (ch >> 1) * PITCH;
    // a few rows at a time, the next ones on their way meanwhile
    const long long stride = half ? a.v_stride : a.k_stride;
    const __nv_bfloat16* const rows = (half ? a.v : a.k) + (long long)(e.w + pos0 - e.y) * stride + h * (NG * KV4_GROUP) + ch * 16;
    auto rows_of = [&](int it, uint4 (&raw)[2]) {
        const int key = it * ROWS + sub;
        raw[0] = raw[1] = make_uint4(0, 0, 0, 0);
        if (sub < ROWS && key >= from && key < to) {
            raw[0] = __ldcg(reinterpret_cast<const uint4*>(rows + key * stride));
            raw[1] = __ldcg(reinterpret_cast<const uint4*>(rows + key * stride) + 1);
        }
    };
    uint4 next[2];
    rows_of(from / ROWS, next);
    {
#pragma unroll 1
        for (int it = from / ROWS; it * ROWS < to; ++it) {
            const uint4 raw[2] = {next[0], next[1]};
            rows_of(it + 1, next);
            const int key = it * ROWS + sub;
            uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
            __nv_bfloat162 least = *reinterpret_cast<const __nv_bfloat162*>(&w[0]), most = least;
#pragma unroll
            for (int j = 1; j < 8; ++j) {
                const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w[j]);
                least = __hmin2(least, v);
                most = __hmax2_nan(most, v);
            }
            float low = fminf(__low2float(least), __high2float(least)), high = __low2float(most);
            high = high <= __high2float(most) ? __high2float(most) : high;       // NaN stays if it is in the first
            const bool odd = !(high <= KV4_LIMIT) || !(low >= -KV4_LIMIT) || __hisnan(__high2bfloat16(most));
            if (odd) {                                                           // so that what is stored is finite
                atomicOr(a.c.flag, KV4_BAD_VALUE);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float x = tame(element(w, j));
                    low = j ? fminf(low, x) : x;
                    high = j ? fmaxf(high, x) : x;
                }
            }
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 1));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
            const __half zero = __float2half_rn(low);
            const float z = __half2float(zero);
            const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(high, z), 1.f / 15.f));
            const float s = __half2float(scale), inv = s > 0.f ? __fdividef(1.f, 15.f * s) : 0.f;
            uint32_t code[16];      // in the low bits of 2^23 + code
            float near = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float q = __saturatef((element(w, j) - z) * inv), c = fmaf(q, 15.f, 8388608.f);
                near = fmaxf(near, fabsf(fmaf(q, 15.f, 8388608.f - c)));
                code[j] = __float_as_uint(c);
            }
            if (near > NEAR || odd) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float f = (odd ? tame(element(w, j)) : element(w, j)) - z, q = __saturatef(f * inv);
                    float c = fmaf(q, 15.f, 8388608.f);
                    if (fabsf(fmaf(q, 15.f, 8388608.f - c)) > NEAR) c = 8388608.f + code_between(f, s, floorf(q * 15.f));
                    code[j] = __float_as_uint(c);
                }
            }
            if (sub >= ROWS || key < from || key >= to) continue;
            const int key8 = key & 7, upper = key >> 3;
            constexpr uint32_t BASE = 0x4B000000u;      // the bits of 2^23
            if (!half) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t word = 0u - BASE * 0x11111111u;
#pragma unroll
                    for (int j = 0; j < 8; ++j) word += code[8 * q + j] << (4 * (j >> 1) + 16 * (j & 1));
                    *reinterpret_cast<uint32_t*>(gimg + (key8 * 4 + (ch & 1) * 2 + q) * 8 + upper * 4) = word;
                }
                if (!(ch & 1)) *reinterpret_cast<__half2*>(gimg + KV4_KPAR + key8 * 8 + upper * 4) = __halves2half2(scale, zero);
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    gimg[(((ch & 1) * 4 + (q >> 1)) * 4 + (key8 >> 1)) * 8 + (q & 1) * 4 + (key8 & 1) * 2 + upper] =
                        (unsigned char)(code[2 * q] + (code[2 * q + 1] << 4));
                if (!(ch & 1)) *reinterpret_cast<__half2*>(gimg + KV4_KPAR + key8 * 8 + upper * 4) = __halves2half2(scale, zero);
            }
        }
    }
    __syncwarp();
    constexpr int SIDE = KV4_GT / 2;           // bytes of a group's keys, and of its values
    unsigned char* const out = tile + (half ? SIDE : 0);
    if (to - from == 16) {
        for (int i = lane; i < NG * (SIDE / 16); i += 32)
            *reinterpret_cast<uint4*>(out + i / (SIDE / 16) * KV4_GT + i % (SIDE / 16) * 16) =
                *reinterpret_cast<const uint4*>(img + i / (SIDE / 16) * PITCH + i % (SIDE / 16) * 16);
        return;
    }
    for (int i = lane; i < NG * (SIDE / 4); i += 32) {      // word i: whose is it?
        const int in = i * 4 % SIDE;
        const unsigned char* const from_img = img + i / (SIDE / 4) * PITCH + in;
        unsigned char* const to_pool = out + i / (SIDE / 4) * KV4_GT + in;
        if (!half || in >= KV4_KPAR) {              // one key's
            const int key = (in < KV4_KPAR ? in >> 5 : (in - KV4_KPAR) >> 3) + (in >> 2 & 1) * 8;
            if (key >= from && key < to) *reinterpret_cast<uint32_t*>(to_pool) = *reinterpret_cast<const uint32_t*>(from_img);
        } else {                                    // four keys', a byte each
            const int key = (in >> 3 & 3) * 2;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = key + (q >> 1) + (q & 1) * 8;
                if (k >= from && k < to) to_pool[q] = from_img[q];
            }
        }
    }
}

// The reverse: 8 elements of four kv heads a thread, bf16 out.  Rows whose slot is out of range or whose position lies behind the sequence's end come out as
// zeros.  A CTA takes the rows next to one another, keys or values (blockIdx.z), because those of a tile share its lines in
// the L1; that is why this kernel starts only when the kernel before it has ended (no early launch: an SM's L1 could hold older lines).
// 16000 rows of 8 heads of 128: 25 us (20 MB in and 65 out: 13 us); with one head a thread, which looks its row up for 8 elements, 29.
constexpr int KV4_READ_HEADS = 4;
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_read(const Kv4RowsArgs a) {
    constexpr int CH = NG * 4, ROWS = 256 / CH;
    const bool value = blockIdx.z != 0;
    const int ch = threadIdx.x % CH, h0 = blockIdx.y * KV4_READ_HEADS;
    const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / CH;
    if (threadIdx.x >= ROWS * CH || row >= a.n_rows) return;
    const int slot = __ldg(a.row_slot + row), pos = __ldg(a.row_pos + row);
    long long where = -1;
    if (slot >= 0 && slot < a.c.max_seqs && pos >= 0 && (pos >> a.c.block_shift) < a.c.max_blocks) {
        const int b = __ldg(a.c.table + (size_t)slot * a.c.max_blocks + (pos >> a.c.block_shift)), len = __ldg(a.c.lens + slot);
        // behind the end lies what the block's last owner stored
        if (b >= 0 && b < a.c.n_blocks && pos < len) where = ((long long)b << a.c.block_shift) + (pos & ((1 << a.c.block_shift) - 1));
    }
    if (where < 0 && slot != -1) atomicOr(a.c.flag, KV4_BAD_SLOT);
    const int key = (int)(where & 15), key8 = key & 7, upper = key >> 3, grp = ch >> 2, t = ch & 3, heads = min(a.c.n_kv - h0, KV4_READ_HEADS);
    const int skip = NG * KV4_GT << (a.c.block_shift - 4);      // from a head to the next in a block
    const unsigned char* const tile = a.c.pool + (where >= 0 ? tile_at<NG>(a.c, where, h0) + grp * KV4_GT : 0);
    uint32_t par[KV4_READ_HEADS];
    uint2 code[KV4_READ_HEADS];
#pragma unroll
    for (int i = 0; i < KV4_READ_HEADS; ++i) {
        par[i] = 0;
        code[i] = make_uint2(0, 0);
        if (where < 0 || i >= heads) continue;
        const unsigned char* const at = tile + i * skip;
        par[i] = __ldg(reinterpret_cast<const uint32_t*>(at + (value ? KV4_VPAR : KV4_KPAR) + key8 * 8 + upper * 4));
        if (!value) {
            code[i].x = __ldg(reinterpret_cast<const uint32_t*>(at + (key8 * 4 + t) * 8 + upper * 4));
        } else {      // the key's bytes of two words each
            const uint2 lo = __ldg(reinterpret_cast<const uint2*>(at + KV4_VCODE + (2 * t * 4 + (key8 >> 1)) * 8));
            const uint2 hi = __ldg(reinterpret_cast<const uint2*>(at + KV4_VCODE + ((2 * t + 1) * 4 + (key8 >> 1)) * 8));
            const unsigned in = (key8 & 1) * 2 + upper, two = in | in + 4 << 4;
            code[i] = make_uint2(__byte_perm(lo.x, lo.y, two), __byte_perm(hi.x, hi.y, two));
        }
    }
    const __half2 unit = __halves2half2(__ushort_as_half(0x3C00), __ushort_as_half(0x2C00));      // 1, 1 / 16
    const __half2 less = __halves2half2(__ushort_as_half(0xE400), __ushort_as_half(0xD400));      // -1024, -64
    __nv_bfloat16* dst = (value ? a.v_out + row * a.v_stride : a.k_out + row * a.k_stride) + (size_t)h0 * (NG * KV4_GROUP) + ch * 8;
#pragma unroll
    for (int i = 0; i < KV4_READ_HEADS; ++i) {
        if (i >= heads) break;
        // pairs of codes as 1024 + c and 1024 + 16 c (a nibble, and one four bits higher, under the exponent of 1024), exact in f16
        uint32_t pair[4], w[4];
        if (!value) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = code[i].x >> (4 * j);
                pair[j] = (two & 0xfu) | (two & 0xf0000u) << 4 | 0x64006400u;      // the odd element four bits higher
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)      // a byte holds both codes of a pair
                pair[j] = (__byte_perm(j < 2 ? code[i].x : code[i].y, 0, j & 1 ? 0x4141 : 0x4040) & 0x00f0000fu) | 0x64006400u;
        }
        const __half2 sz = *reinterpret_cast<const __half2*>(&par[i]), s = __low2half2(sz), z = __high2half2(sz);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 c = __hfma2(*reinterpret_cast<const __half2*>(&pair[j]), unit, less), v = __hfma2(s, c, z);
            const __nv_bfloat162 p = __floats2bfloat162_rn(__low2float(v), __high2float(v));
            w[j] = *reinterpret_cast<const uint32_t*>(&p);
        }
        *reinterpret_cast<uint4*>(dst + i * (NG * KV4_GROUP)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace vuik
