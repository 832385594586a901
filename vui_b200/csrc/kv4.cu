// Host side of the paged 4-bit KV cache: checks, sizes and launches (kernels: kv4_kernels.cuh, kv4_attn.cuh).  Entry points:
// include/vuib200.h, section "Paged KV cache in 4 bits".
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <new>

#include "../../include/vuib200.h"
#include "kv4_attn.cuh"
#include "kv4_kernels.cuh"

using namespace vuik;

struct VuibKv4 {
    VuibKv4Config cfg;
    Kv4Cache cache;           // pool: of layer 0
    size_t layer_bytes;
    bool bound;
    int block_shift, ng, sms, device;
    int resident[5];          // CTAs of each attention form that fit an SM of the device, 0: not asked for yet
    int64_t launches;
    char err[256];
};

namespace {

int32_t fail(VuibKv4* c, int32_t code, const char* fmt, ...) {
    if (c) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(c->err, sizeof(c->err), fmt, ap);
        va_end(ap);
    }
    return code;
}

#define CK(call)                                                                              \
    do {                                                                                      \
        cudaError_t _err = (call);                                                            \
        if (_err != cudaSuccess)                                                              \
            return fail(c, VUIB_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(_err));  \
    } while (0)

// cluster 0: without an early launch
template <class... KArgs, class... Args>
cudaError_t launch(VuibKv4* c, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, void* stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : cluster;
    c->launches++;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// What a plan's shape decides for attention: the form, the columns of a tile (rows x query heads of a kv head) and the positions of a split.
//   FEW_2, FEW_4   bytes: up to 2 columns (heads of 64 and 128) and up to 4.  256 sequences of 512 to 2048 positions, two query heads a kv head of 64:
//                  53 us with FEW_2, 64 with FEW_4, 105 with MANY_16; 4 query heads of 128, 4 x 64k positions: 77 with FEW_4, 92 with MANY_8.
//   MANY_8, _16    f16, a warp's own keys: up to 8 and 16 columns a tile.  64 sequences of 800 to 4000, 8 query heads a kv head of 128 (8 kv heads): 71 us
//                  with MANY_8, 91 with MANY_16; 16 query heads (4 kv heads): 69 and 57; tiles of 32 columns, when they were built, were
//                  slower wherever they fill (64 x 24 rows of 2 query heads of 64: 30 us with 16, 45 with 32).
//   ROWS           f16, shared keys, 128 columns: from 128 columns of heads of 128 on, 256 of 64, 512 of 96.  Against MANY_16, us: heads of 128, 128
//                  columns 28 and 29, 256 32 and 47, 2 x 1000 rows 1060 and 1556; heads of 64, 128 columns 38 and 32, 256 43 and 55, 2000 38 and
//                  40; heads of 96, 300 columns 39 and 32, 600 54 and 54.
// Splits.  Up to 16 columns by the sequence's length alone, so that a row's bits do not depend on what else is there: one of up to 512 positions is one
// piece (64 sequences of 64 to 512: 10.4 us, in pieces of 256 12.9), up to 1024 pieces of 256 (16 sequences of 600 to 1000, 8 query heads a kv head of
// 128: 12.5, in pieces of 512 15.7), beyond of 512 (4 x 64k: 77, 256 82, 1024 80).  More columns: none where the tiles fill the SMs, else pieces of 512,
// at most 8 of a sequence, so that their sums stay a few megabytes.
enum Form { FEW_2, FEW_4, MANY_8, MANY_16, ROWS };
struct Shape { Form form; int cols; Kv4Split split; };
Shape shape_of(const VuibKv4* c, const VuibKv4Plan* p) {
    const int group = c->cfg.n_heads / c->cfg.n_kv_heads;
    const long long most = (long long)p->max_new * group;       // columns of one sequence
    const int rows_from = c->ng == 4 ? 128 : c->ng == 3 ? 512 : 256;
    const Form form = most <= 2 && c->ng != 3 ? FEW_2 : most <= 4 ? FEW_4 : most <= 8 ? MANY_8 : most < rows_from ? MANY_16 : ROWS;
    const int cols = form == FEW_2 ? 2 : form == FEW_4 ? 4 : form == MANY_8 ? 8 : form == MANY_16 ? 16 : KR_COLS;
    if (most <= 16) return {form, cols, {512, 256, 512, 1 << 30, true}};
    const long long tiles = ceil_div((long long)p->n_rows * group, cols) + p->n_seqs;
    const long long len = (long long)c->cfg.max_blocks << c->block_shift;
    const int split = tiles * c->cfg.n_kv_heads >= 2 * c->sms ? 1 << 30 : 512;
    return {form, cols, {split, split, split, 8, tiles * (len / 64 + 16) < KV4_MANY}};
}

// Most splits of one sequence.
long long most_parts(const VuibKv4* c, const Shape& s) {
    const long long len = (long long)c->cfg.max_blocks << c->block_shift;
    return min((long long)s.split.most, max(ceil_div(min(len, 512ll), s.split.up_to_512),
                                            max(len > 512 ? ceil_div(min(len, 1024ll), s.split.up_to_1024) : 0, ceil_div(len, s.split.beyond))));
}

// Most units (of one kv head) that a plan of this shape can have.  Sequences share no blocks, so their lengths sum up to the pool's.
long long most_units(const VuibKv4* c, const VuibKv4Plan* p, const Shape& s) {
    const long long pool = (long long)c->cfg.n_blocks << c->block_shift;
    const int group = c->cfg.n_heads / c->cfg.n_kv_heads;
    const long long a_seq = ceil_div((long long)p->max_new * group, s.cols);
    const long long tiles = min((long long)p->n_seqs * a_seq, ceil_div((long long)p->n_rows * group, s.cols) + p->n_seqs);
    return min(tiles * most_parts(c, s), a_seq * (p->n_seqs + pool / min(s.split.up_to_512, s.split.up_to_1024)));
}

// Units whose sums may have to be kept.
long long most_items(const VuibKv4* c, const VuibKv4Plan* p, const Shape& s) { return most_units(c, p, s) * c->cfg.n_kv_heads; }

size_t acc_bytes(const VuibKv4* c, long long items, int cols) { return ((size_t)items * cols * c->cfg.head_dim * 4 + 255) & ~size_t(255); }

// Shared memory of the plan's kernel.
size_t plan_smem(int n_seqs, int max_seqs) { return (8 * (size_t)n_seqs + 3 + max_seqs) * 4; }

// The parts of a plan's work array.
int4* plan_entries(const VuibKv4Plan* p) { return reinterpret_cast<int4*>(p->work); }
int32_t* plan_units(const VuibKv4Plan* p) { return p->work + 4 * (size_t)p->n_seqs; }
int32_t* plan_work(const VuibKv4Plan* p) { return p->work + 5 * (size_t)p->n_seqs + 1; }
int32_t* plan_tiles(const VuibKv4Plan* p) { return p->work + 6 * (size_t)p->n_seqs + 2; }
int32_t* plan_row_entry(const VuibKv4Plan* p) { return p->work + 7 * (size_t)p->n_seqs + 3; }

int32_t check_plan(VuibKv4* c, const VuibKv4Plan* p) {
    if (!p || !p->work || !p->cu_rows) return fail(c, VUIB_ERR_NULL, "a plan needs its arrays");
    if (p->n_rows > 0 && (!p->row_slot || !p->row_pos || !p->slot_map)) return fail(c, VUIB_ERR_NULL, "a plan of rows needs its row arrays");
    if (p->n_seqs < 1 || p->n_seqs > KV4_MAX_SEQS) return fail(c, VUIB_ERR_RANGE, "n_seqs %d not in 1..%d", p->n_seqs, KV4_MAX_SEQS);
    if (p->n_rows < 0 || p->n_rows > 1 << 24) return fail(c, VUIB_ERR_RANGE, "n_rows %d not in 0..%d", p->n_rows, 1 << 24);
    if (p->max_new < 0 || p->max_new > p->n_rows) return fail(c, VUIB_ERR_RANGE, "max_new %d not in 0..n_rows", p->max_new);
    if (reinterpret_cast<uintptr_t>(p->work) & 15) return fail(c, VUIB_ERR_WORKSPACE, "work must be 16-byte aligned");
    if (!c->bound) return fail(c, VUIB_ERR_UNBOUND, "vuib_kv4_bind has not been called");
    return VUIB_OK;
}

// A matrix of rows: 16-byte aligned, rows at a multiple of 8 elements and not overlapping.
int32_t check_rows(VuibKv4* c, const char* name, const void* p, int64_t stride, int64_t width) {
    if (!p) return fail(c, VUIB_ERR_NULL, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) & 15 || stride % 8 || stride < width)
        return fail(c, VUIB_ERR_SHAPE, "%s: rows must be 16-byte aligned, a multiple of 8 elements and at least %lld apart (stride %lld)", name,
                    (long long)width, (long long)stride);
    return VUIB_OK;
}

template <int NG>
cudaError_t launch_attn(VuibKv4* c, const Shape& s, void (*kern)(Kv4AttnArgs), int threads, int smem, Kv4AttnArgs a, long long items, bool merge, void* stream) {
    int& resident = c->resident[s.form];
    cudaError_t e = cudaSuccess;
    if (!resident) {     // as many CTAs as fit the SMs: asked for, and attributes set, once a handle and form
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kern, threads, smem);
        if (e != cudaSuccess) return e;
        if (resident < 1) resident = 1;
    }
    const long long room = (long long)c->sms * resident;
    // A kernel that starts beside the merge finds its SMs partly taken, and one that fills them all then has late CTAs: 256 sequences of
    // 512 to 2048 positions call after call 61.7 us with an early start and 53.4 without, one sequence of 1300 7.8 and 7.9.
    a.early = 2 * items < room;
    const long long grid = min(items, room), rows = (long long)a.n_rows * c->cfg.n_heads;
    e = launch(c, kern, dim3((unsigned)grid), threads, smem, 1, stream, a);
    if (e != cudaSuccess || !merge) return e;
    if (most_parts(c, s) <= 32)
        return launch(c, k_kv4_merge<NG, 1>, dim3((unsigned)ceil_div(rows, 4)), 128, 0, 1, stream, a, s.cols);
    return launch(c, k_kv4_merge<NG, 8>, dim3((unsigned)rows), 256, 0, 1, stream, a, s.cols);
}

template <int NG>
cudaError_t launch_form(VuibKv4* c, const Shape& s, const Kv4AttnArgs& a, long long items, bool merge, void* stream) {
    constexpr int T = KA_THREADS + 32;
    switch (s.form) {
        case FEW_2:
            if constexpr (NG != 3) return launch_attn<NG>(c, s, k_kv4_attn_few<NG, true>, T, KaShared<NG, 2>::TOTAL, a, items, merge, stream);
        case FEW_4: return launch_attn<NG>(c, s, k_kv4_attn_few<NG, false>, T, KaShared<NG, 4>::TOTAL, a, items, merge, stream);
        case MANY_8: return launch_attn<NG>(c, s, k_kv4_attn<NG, 1>, T, KaShared<NG, 8>::TOTAL, a, items, merge, stream);
        case ROWS: return launch_attn<NG>(c, s, k_kv4_attn_rows<NG>, KR_THREADS, KrShared<NG>::TOTAL, a, items, merge, stream);
        default: return launch_attn<NG>(c, s, k_kv4_attn<NG, 2>, T, KaShared<NG, 16>::TOTAL, a, items, merge, stream);
    }
}

}  // namespace

extern "C" int32_t vuib_kv4_create(const VuibKv4Config* cfg, VuibKv4** out) {
    if (!cfg || !out) return VUIB_ERR_NULL;
    *out = nullptr;
    const VuibKv4Config& g = *cfg;
    if (g.head_dim != 64 && g.head_dim != 96 && g.head_dim != 128) return VUIB_ERR_SHAPE;
    if (g.n_kv_heads < 1 || g.n_heads < g.n_kv_heads || g.n_heads % g.n_kv_heads || g.n_heads / g.n_kv_heads > 16 || g.n_heads > 1024)
        return VUIB_ERR_SHAPE;
    int shift = 4;
    while (shift < 8 && 1 << shift < g.block_size) ++shift;
    if (1 << shift != g.block_size) return VUIB_ERR_SHAPE;
    if (g.n_layers < 1 || g.n_layers > 1024 || g.n_blocks < 1 || g.n_blocks > 1 << 24 || g.max_seqs < 1 || g.max_seqs > KV4_MAX_SEQS ||
        g.max_blocks < 1 || (long long)g.max_blocks << shift > 1 << 24)
        return VUIB_ERR_RANGE;
    VuibKv4* c = new (std::nothrow) VuibKv4();
    if (!c) return VUIB_ERR_NULL;
    memset(c, 0, sizeof(*c));
    c->cfg = g;
    c->block_shift = shift;
    c->ng = g.head_dim / KV4_GROUP;
    c->layer_bytes = (size_t)g.n_blocks * g.n_kv_heads * (g.block_size / KV4_TILE) * c->ng * KV4_GT;
    *out = c;
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_destroy(VuibKv4* c) {
    delete c;
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_last_error(VuibKv4* c, char* buf, size_t n) {
    if (!c || !buf || !n) return VUIB_ERR_NULL;
    snprintf(buf, n, "%s", c->err);
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_pool_bytes(VuibKv4* c, size_t* bytes) {
    if (!c || !bytes) return VUIB_ERR_NULL;
    *bytes = c->layer_bytes * c->cfg.n_layers;
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_bind(VuibKv4* c, void* pool, size_t bytes, int32_t* seq_lens, int32_t* block_table, int32_t* free_blocks,
                                 int32_t* n_free, int32_t* flag) {
    if (!c) return VUIB_ERR_NULL;
    c->bound = false;
    if (!pool || !seq_lens || !block_table || !free_blocks || !n_free || !flag) return fail(c, VUIB_ERR_NULL, "a pointer is NULL");
    if (reinterpret_cast<uintptr_t>(pool) & 127) return fail(c, VUIB_ERR_WORKSPACE, "the pool must be 128-byte aligned");
    if (bytes < c->layer_bytes * c->cfg.n_layers)
        return fail(c, VUIB_ERR_WORKSPACE, "pool of %zu bytes, %zu needed", bytes, c->layer_bytes * c->cfg.n_layers);
    memset(c->resident, 0, sizeof(c->resident));
    CK(cudaGetDevice(&c->device));
    CK(cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, c->device));
    // For the largest plan there can be: the attribute is the kernel's, not a call's, and what a launch gets without it holds the kernel's
    // static arrays too.
    CK(cudaFuncSetAttribute(k_kv4_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem(KV4_MAX_SEQS, KV4_MAX_SEQS)));
    c->cache = {static_cast<unsigned char*>(pool), block_table, seq_lens, free_blocks, n_free, flag, c->cfg.n_kv_heads, c->block_shift,
                c->cfg.n_blocks, c->cfg.max_seqs, c->cfg.max_blocks};
    c->bound = true;
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_reset(VuibKv4* c, void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (!c->bound) return fail(c, VUIB_ERR_UNBOUND, "vuib_kv4_bind has not been called");
    const long long n = (long long)c->cfg.max_seqs * c->cfg.max_blocks;
    CK(launch(c, k_kv4_reset, dim3((unsigned)min(ceil_div(max(n, (long long)c->cfg.n_blocks), 256), 1024ll)), 256, 0, 1, stream, c->cache));
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_plan(VuibKv4* c, const VuibKv4Plan* p, const int32_t* slots_dev, const int32_t* new_dev, const int32_t* at_dev,
                                 void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (int32_t rc = check_plan(c, p)) return rc;
    if (!slots_dev) return fail(c, VUIB_ERR_NULL, "slots is NULL");
    if (!new_dev && p->max_new < 1) return fail(c, VUIB_ERR_RANGE, "one new row each, but max_new is %d", p->max_new);
    const Shape s = shape_of(c, p);
    if (most_units(c, p, s) >= KV4_MANY) return fail(c, VUIB_ERR_RANGE, "too many units of work for one plan");
    Kv4PlanArgs a = {};
    a.c = c->cache;
    a.slots = slots_dev; a.new_lens = new_dev; a.at = at_dev;
    a.n = p->n_seqs; a.n_rows = p->n_rows; a.max_new = p->max_new;
    a.group = c->cfg.n_heads / c->cfg.n_kv_heads; a.cols = s.cols; a.split = s.split;
    a.entries = plan_entries(p); a.cu_units = plan_units(p); a.cu_work = plan_work(p); a.cu_tiles = plan_tiles(p); a.row_entry = plan_row_entry(p);
    a.cu_rows = p->cu_rows;
    a.row_slot = p->row_slot; a.row_pos = p->row_pos; a.slot_map = reinterpret_cast<long long*>(p->slot_map);
    const size_t smem = plan_smem(p->n_seqs, c->cfg.max_seqs);
    // One CTA where little is written: a cluster's barriers cost 2 us.  Rows are known here; cut-backs can give back any number of blocks.
    const int cluster = p->n_rows > 4096 || (at_dev && p->n_seqs > 64 && c->cfg.n_blocks > 4096) ? 8 : 1;
    const int threads = p->n_seqs <= 256 && p->n_rows <= 1024 ? 256 : 1024;
    CK(launch(c, k_kv4_plan, dim3(cluster), threads, smem, cluster, stream, a));
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_append(VuibKv4* c, int32_t layer, const VuibKv4Plan* p, const void* k_dev, int64_t k_stride, const void* v_dev,
                                   int64_t v_stride, void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (int32_t rc = check_plan(c, p)) return rc;
    if (layer < 0 || layer >= c->cfg.n_layers) return fail(c, VUIB_ERR_RANGE, "layer %d not in 0..%d", layer, c->cfg.n_layers - 1);
    if (!p->n_rows) return VUIB_OK;
    const int64_t width = (int64_t)c->cfg.n_kv_heads * c->cfg.head_dim;
    if (int32_t rc = check_rows(c, "k", k_dev, k_stride, width)) return rc;
    if (int32_t rc = check_rows(c, "v", v_dev, v_stride, width)) return rc;
    Kv4RowsArgs a = {};
    a.c = c->cache;
    a.c.pool += c->layer_bytes * layer;
    a.k = static_cast<const __nv_bfloat16*>(k_dev); a.k_stride = k_stride;
    a.v = static_cast<const __nv_bfloat16*>(v_dev); a.v_stride = v_stride;
    a.entries = plan_entries(p); a.cu_tiles = plan_tiles(p); a.n = p->n_seqs;
    a.n_rows = p->n_rows;
    // a sequence's m rows touch (m + 30) / 16 tiles at most, and no more than m
    const long long tiles = min((long long)p->n_rows, p->n_rows / 16 + 2ll * p->n_seqs);
    const dim3 grid((unsigned)ceil_div(tiles * c->cfg.n_kv_heads, 4), 2);
    CK(c->ng == 2 ? launch(c, k_kv4_append<2>, grid, 128, 0, 1, stream, a)
                  : c->ng == 3 ? launch(c, k_kv4_append<3>, grid, 128, 0, 1, stream, a) : launch(c, k_kv4_append<4>, grid, 128, 0, 1, stream, a));
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_read(VuibKv4* c, int32_t layer, int32_t n_rows, const int32_t* row_slot_dev, const int32_t* row_pos_dev,
                                 void* k_out_dev, int64_t k_stride, void* v_out_dev, int64_t v_stride, void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (!c->bound) return fail(c, VUIB_ERR_UNBOUND, "vuib_kv4_bind has not been called");
    if (layer < 0 || layer >= c->cfg.n_layers) return fail(c, VUIB_ERR_RANGE, "layer %d not in 0..%d", layer, c->cfg.n_layers - 1);
    if (n_rows < 0 || n_rows > 1 << 24) return fail(c, VUIB_ERR_RANGE, "n_rows %d not in 0..%d", n_rows, 1 << 24);
    if (!n_rows) return VUIB_OK;
    if (!row_slot_dev || !row_pos_dev) return fail(c, VUIB_ERR_NULL, "row_slot or row_pos is NULL");
    const int64_t width = (int64_t)c->cfg.n_kv_heads * c->cfg.head_dim;
    if (int32_t rc = check_rows(c, "k_out", k_out_dev, k_stride, width)) return rc;
    if (int32_t rc = check_rows(c, "v_out", v_out_dev, v_stride, width)) return rc;
    Kv4RowsArgs a = {};
    a.c = c->cache;
    a.c.pool += c->layer_bytes * layer;
    a.k_out = static_cast<__nv_bfloat16*>(k_out_dev); a.k_stride = k_stride;
    a.v_out = static_cast<__nv_bfloat16*>(v_out_dev); a.v_stride = v_stride;
    a.row_slot = row_slot_dev; a.row_pos = row_pos_dev;
    a.n_rows = n_rows;
    const dim3 grid((unsigned)ceil_div(n_rows, 256 / (c->ng * 4)), (unsigned)ceil_div(c->cfg.n_kv_heads, KV4_READ_HEADS), 2);
    CK(c->ng == 2 ? launch(c, k_kv4_read<2>, grid, 256, 0, 0, stream, a)
                  : c->ng == 3 ? launch(c, k_kv4_read<3>, grid, 256, 0, 0, stream, a) : launch(c, k_kv4_read<4>, grid, 256, 0, 0, stream, a));
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_attention_workspace(VuibKv4* c, const VuibKv4Plan* p, size_t* bytes) {
    if (!c || !bytes) return VUIB_ERR_NULL;
    if (int32_t rc = check_plan(c, p)) return rc;
    *bytes = 0;
    if (!p->n_rows || !p->max_new) return VUIB_OK;
    const Shape s = shape_of(c, p);
    if (most_parts(c, s) <= 1) return VUIB_OK;
    const long long items = most_items(c, p, s);
    *bytes = acc_bytes(c, items, s.cols) + (size_t)items * s.cols * 8;
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_attention(VuibKv4* c, int32_t layer, const VuibKv4Plan* p, const void* q_dev, int64_t q_stride, void* out_dev,
                                      int64_t out_stride, float scale, void* ws_dev, size_t ws_bytes, void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (int32_t rc = check_plan(c, p)) return rc;
    if (layer < 0 || layer >= c->cfg.n_layers) return fail(c, VUIB_ERR_RANGE, "layer %d not in 0..%d", layer, c->cfg.n_layers - 1);
    if (!(scale >= 0.f) || scale > 1e30f) return fail(c, VUIB_ERR_RANGE, "scale must be positive, or 0 for 1/sqrt(head_dim)");
    if (!p->n_rows || !p->max_new) return VUIB_OK;
    const int64_t width = (int64_t)c->cfg.n_heads * c->cfg.head_dim;
    if (int32_t rc = check_rows(c, "q", q_dev, q_stride, width)) return rc;
    if (int32_t rc = check_rows(c, "out", out_dev, out_stride, width)) return rc;
    size_t need = 0;
    if (int32_t rc = vuib_kv4_attention_workspace(c, p, &need)) return rc;
    if (need && (!ws_dev || ws_bytes < need || reinterpret_cast<uintptr_t>(ws_dev) & 255))
        return fail(c, VUIB_ERR_WORKSPACE, "workspace of %zu bytes, 256-byte aligned, needed", need);
    const Shape s = shape_of(c, p);
    const long long items = most_items(c, p, s);
    Kv4AttnArgs a = {};
    a.c = c->cache;
    a.c.pool += c->layer_bytes * layer;
    a.entries = plan_entries(p); a.cu_units = plan_units(p); a.cu_work = plan_work(p); a.row_entry = plan_row_entry(p);
    a.n = p->n_seqs; a.n_rows = p->n_rows; a.group = c->cfg.n_heads / c->cfg.n_kv_heads; a.split = s.split;
    a.group_inv = a.group > 1 ? (uint32_t)(((1ull << 32) + a.group - 1) / a.group) : 0;
    a.q = static_cast<const __nv_bfloat16*>(q_dev); a.q_stride = q_stride;
    a.out = static_cast<__nv_bfloat16*>(out_dev); a.out_stride = out_stride;
    a.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)c->cfg.head_dim)) * 1.4426950408889634f;
    a.acc = static_cast<float*>(ws_dev);
    a.ml = reinterpret_cast<float2*>(static_cast<char*>(ws_dev) + acc_bytes(c, items, s.cols));
    const bool merge = need != 0;
    CK(c->ng == 2 ? launch_form<2>(c, s, a, items, merge, stream)
                  : c->ng == 3 ? launch_form<3>(c, s, a, items, merge, stream) : launch_form<4>(c, s, a, items, merge, stream));
    return VUIB_OK;
}

extern "C" int32_t vuib_kv4_check_flag(VuibKv4* c, void* stream) {
    if (!c) return VUIB_ERR_NULL;
    if (!c->bound) return fail(c, VUIB_ERR_UNBOUND, "vuib_kv4_bind has not been called");
    int32_t v = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    CK(cudaMemcpyAsync(&v, c->cache.flag, 4, cudaMemcpyDeviceToHost, s));
    CK(cudaStreamSynchronize(s));
    if (!v) return VUIB_OK;
    CK(cudaMemsetAsync(c->cache.flag, 0, 4, s));
    return fail(c, VUIB_ERR_DEVICE_FLAG, "device flag %d:%s%s%s%s%s%s%s", v, v & KV4_BAD_SLOT ? " slot or position out of range or named twice;" : "",
                v & KV4_BAD_LEN ? " length out of range;" : "", v & KV4_NO_ROWS ? " more rows than the plan holds;" : "",
                v & KV4_NO_BLOCKS ? " out of blocks;" : "", v & KV4_BAD_VALUE ? " NaN or a value beyond 60000 stored;" : "",
                v & KV4_BAD_BLOCK ? " no block for a position;" : "", v & KV4_TIMEOUT ? " a wait inside a kernel ran out;" : "");
}

extern "C" int64_t vuib_kv4_launch_count(VuibKv4* c) { return c ? c->launches : 0; }
