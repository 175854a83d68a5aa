// C ABI of tree attention and of the rows and pages of a paged cache (declared
// in include/voltattn.h): argument checks, workspace layout and launch.
#include <algorithm>
#include <cmath>
#include <climits>
#include <initializer_list>

#include "../../include/voltattn.h"
#include "cache_rows.cuh"
#include "decode_tree.cuh"
#include "launch.cuh"
#include "pages.cuh"

using namespace va;
using namespace va::host;

namespace {

constexpr int kMaxNodes = 64;
constexpr int kMaxSplits = kTreeMaxSplits;
constexpr int kMaxForks = 4000;
// Rows of a table in decode_tree: positions are 32-bit, and rounding a range up to whole blocks and
// parts adds less than 2^16 to them.
constexpr long long kMaxTreeRows = (long long)INT_MAX - (1 << 16);

bool pool_fmt(int f) { return f >= VA_F16 && f < VA_Q4CP; }
bool tree_fmt(int f) {
    return f == VA_F16P || f == VA_BF16P || f == VA_F8P || f == VA_Q8P || f == VA_Q4P || f == VA_Q3P;
}
bool has_scales(int f) { return f != VA_F16 && f != VA_F16P && f != VA_BF16P; }
bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool all_aligned4(std::initializer_list<const void*> ps) {
    return std::all_of(ps.begin(), ps.end(), [](const void* p) { return aligned_to(p, 4); });
}
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Checks of what every entry point here takes: the pool's shape and its buffers.
int check_pool(int fmt, const va_bufs* b, int B, int max_pages, int Hkv, int page_rows, int num_pages, int D) {
    if (fmt < VA_F16 || fmt > VA_Q4CP || !b) return VA_ERR_INVALID;
    if (!pool_fmt(fmt) || (D != 64 && D != 128)) return VA_ERR_UNSUPPORTED;
    if (B < 1 || max_pages < 1 || Hkv < 1 || page_rows < 1 || num_pages < 1) return VA_ERR_INVALID;
    if ((long long)max_pages * page_rows > INT_MAX || (long long)B * max_pages > INT_MAX) return VA_ERR_TOO_LARGE;
    if (!b->K || !b->V || (has_scales(fmt) && (!b->scK || !b->scV))) return VA_ERR_INVALID;
    if (!aligned16(b->K) || !aligned16(b->V) || (has_scales(fmt) && (!aligned16(b->scK) || !aligned16(b->scV))))
        return VA_ERR_ALIGN;
    return VA_OK;
}

// Rows of a CTA's tile of query rows: 16 (decode_tree.cuh), 128 or 256 (decode_tree_tc.cuh).
// The large tiles read the cache once for all their rows but cost more to start: 18 us in
// tiles of 16 against 26 in one of 128 (128 query rows, 8 KV heads x 1024 rows, q4+), 43
// against 32 at 4 x 4000 rows. Few live rows leave them idle: 64 rows of q8+, 16
// sequences up to 8192 rows, take 101 us in tiles of 16, 107 in one of 128. fp16 rows go to
// the tensor cores without a conversion: 64 rows 132 against 74 us, 32 rows 88
// against 70. fp8 rows of 128 dims take the longest to convert, so they need more query rows: 80 rows,
// 16 sequences of 1000 to 4000, 127 against 138, 128 rows 185 against 140 (128 with half of them
// live 128 against 138; of 64 dims 80 rows already gain). The sizes are those of the tables, the
// lengths being on the device.
int tree_rows(int fmt, int B, int Hkv, int R, int Lmax, int D) {
    const bool f16 = fmt == VA_F16P;
    const double work = (double)B * Hkv * Lmax * R;
    const int small = f16 ? 16 : fmt == VA_F8P && D == 128 ? 96 : 64;
    if (R <= small || work <= (f16 ? 1 << 21 : 1 << 23)) return 16;
    return R <= 128 ? 128 : 256;
}

// Completion counters, one per (sequence, KV head, row tile), at the front of the
// workspace: a fixed number, so the slots of a call never lie where a call of
// another shape expects zeroed counters. More row tiles than this fill any
// device without splits.
constexpr long long kCounters = 16384;
constexpr size_t kCounterBytes = kCounters * sizeof(unsigned);

// Tiles of 16 rows: the splits with the least cost: the CTAs' rows (of sequences that fill
// 5/8 of their tables on average, plus a CTA's fixed work in rows) shared by the device's
// slots, and half of the longest range for the uneven end; smallest S first. The larger
// tiles' CTAs share the work evenly by themselves: S only has to let the longest
// sequence spread, here one of 2.5 times the mean length. Tables of up to 640 rows are
// not split there: merging two parts takes longer than 5 blocks (2 x 300 rows, f16+, 256
// query rows: 17 us whole, 23 us in parts).
int tree_splits(int nsm, int rows, int B, int Hkv, int R, int Lmax) {
    const double ctas = (double)B * Hkv * ((R + rows - 1) / rows);
    if (ctas > (double)kCounters) return 1;
    const int units = (Lmax + kTreeUnit - 1) / kTreeUnit, most = std::min(kMaxSplits, units);
    if (rows != 16) return most <= 5 ? 1 : std::min(most, (int)std::ceil(2.5 * nsm / ctas) + 1);
    const double load = ctas / (3.0 * nsm), fixed = 320.0;
    double best = 1e300;
    int S = 1;
    for (int s = 1; s <= most && load * s * fixed < best; ++s) {
        const double chunk = (double)((units + s - 1) / s) * kTreeUnit;
        const double cost = std::max(1.0, load * s) * (0.625 * chunk + fixed) + 0.5 * chunk;
        if (cost < best - 1e-9) {
            best = cost;
            S = s;
        }
    }
    return S;
}

// Division by d >= 1 as a multiplication (round-up method): with 2^(l-1) < d <=
// 2^l and m = floor(2^32 (2^l - d) / d) + 1, floor(n / d) = (mulhi(n, m) + n) >> l for
// every n < 2^31.
void divisor(int d, unsigned& mul, unsigned& shift) {
    shift = 0;
    while ((1ll << shift) < d) ++shift;
    mul = (unsigned)((((unsigned long long)1 << 32) * ((1ull << shift) - (unsigned)d)) / (unsigned)d + 1);
}

// A buffer of int32, and whether the first `outs` of some (the outputs) lie in any other of them.
struct Span {
    const int* p;
    long long n;
};
bool outputs_overlap(std::initializer_list<Span> spans, int outs) {
    const Span* s = spans.begin();
    for (int i = 0; i < outs; ++i)
        for (int j = 0; j < (int)spans.size(); ++j) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(s[i].p), b = reinterpret_cast<uintptr_t>(s[j].p);
            if (j != i && a < b + 4 * (uintptr_t)s[j].n && b < a + 4 * (uintptr_t)s[i].n) return true;
        }
    return false;
}

int check_layers(int Hkv, int page_rows, int num_pages, int layers) {
    if (layers < 1) return VA_ERR_INVALID;
    if (layers > 65535 || Hkv > 65535) return VA_ERR_TOO_LARGE;
    if ((long long)layers * num_pages > (1ll << 31) || (long long)Hkv * page_rows > (1ll << 24)) return VA_ERR_TOO_LARGE;
    return VA_OK;
}

PoolView make_pool(int fmt, const va_bufs* b, int Hkv, int page_rows, int num_pages, int D, int layers) {
    PoolView v = {};
    const void* base[4] = {b->K, b->V, b->scK, b->scV};
    for (int i = 0; i < 4; ++i) {
        const bool on = i < 2 || has_scales(fmt);
        v.base[i] = on ? static_cast<uint8_t*>(const_cast<void*>(base[i])) : nullptr;
        v.row_bytes[i] = i < 2 ? (int)va_payload_bytes(fmt, (size_t)D) : 2 * (D / kGroup);
    }
    v.Hkv = Hkv;
    v.page_rows = page_rows;
    v.num_pages = num_pages;
    v.layers = layers;
    return v;
}

}  // namespace

extern "C" {

size_t va_tree_workspace_bytes(int B, int Hq, int Hkv, int Q, int D, int S) {
    if (B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || Q < 1 || Q > kMaxNodes || D < 1 || S < 1 || S > kMaxSplits) return 0;
    const size_t slots = (size_t)B * Hq * Q * S;
    return kCounterBytes + (S > 1 ? round256(slots * 8) + slots * D * sizeof(float) : 0);
}

int va_suggest_tree_splits(int fmt, int B, int Hq, int Hkv, int Q, int Lmax, int D, int* S) {
    if (!S || fmt < VA_F16 || fmt > VA_Q4CP || B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || Q < 1 || Q > kMaxNodes || Lmax < 1)
        return VA_ERR_INVALID;
    if (!tree_fmt(fmt) || (D != 64 && D != 128)) return VA_ERR_UNSUPPORTED;
    int dev;
    const int rc = current_device(&dev);
    if (rc) return rc;
    const int R = Hq / Hkv * Q;
    *S = tree_splits(sm_count(dev), tree_rows(fmt, B, Hkv, R, Lmax, D), B, Hkv, R, Lmax);
    return VA_OK;
}

int va_tree_tile_rows(int fmt, int B, int Hq, int Hkv, int Q, int Lmax, int D, int* rows) {
    if (!rows || fmt < VA_F16 || fmt > VA_Q4CP || B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || Q < 1 || Q > kMaxNodes || Lmax < 1)
        return VA_ERR_INVALID;
    if (!tree_fmt(fmt) || (D != 64 && D != 128)) return VA_ERR_UNSUPPORTED;
    *rows = tree_rows(fmt, B, Hkv, Hq / Hkv * Q, Lmax, D);
    return VA_OK;
}

int va_decode_tree(int fmt, const va_bufs* b, const long long* q_strides, const long long* out_strides,
                   const uint64_t* tree_mask, const int* lens, const int* nodes, const int* block_table, int max_pages,
                   int B, int Hq, int Hkv, int Q, int page_rows, int num_pages, int D, int S, void* ws,
                   size_t ws_bytes, void* stream) {
    int rc = check_pool(fmt, b, B, max_pages, Hkv, page_rows, num_pages, D);
    if (rc) return rc;
    if (!tree_fmt(fmt) || page_rows % 8) return VA_ERR_UNSUPPORTED;
    if (!tree_mask || !lens || !block_table || !b->q || !b->out) return VA_ERR_INVALID;
    if (Hq < 1 || Hq % Hkv || Q < 1 || S < 0) return VA_ERR_INVALID;
    if (Q > kMaxNodes || S > kMaxSplits) return VA_ERR_TOO_LARGE;
    if (!aligned16(b->q) || !aligned_to(b->out, 8)) return VA_ERR_ALIGN;
    if (!aligned_to(tree_mask, 8) || !all_aligned4({lens, nodes, block_table})) return VA_ERR_ALIGN;
    const long long dense[3] = {(long long)Q * Hq * D, (long long)Hq * D, D};
    const long long* qs = q_strides ? q_strides : dense;
    const long long* os = out_strides ? out_strides : dense;
    for (int i = 0; i < 3; ++i)
        if (qs[i] % 8 || os[i] % 8) return VA_ERR_ALIGN;
    if ((long long)max_pages * page_rows > kMaxTreeRows) return VA_ERR_TOO_LARGE;
    if ((long long)B * Hq * Q > INT_MAX / kMaxSplits) return VA_ERR_TOO_LARGE;
    const int R = Hq / Hkv * Q, rows = tree_rows(fmt, B, Hkv, R, max_pages * page_rows, D);
    if (!ws || !aligned16(ws)) return VA_ERR_WORKSPACE;
    if (S == 0) {
        int dev;
        rc = current_device(&dev);
        if (rc) return rc;
        S = tree_splits(sm_count(dev), rows, B, Hkv, R, max_pages * page_rows);
        while (S > 1 && ws_bytes < va_tree_workspace_bytes(B, Hq, Hkv, Q, D, S)) --S;
    }
    if (ws_bytes < va_tree_workspace_bytes(B, Hq, Hkv, Q, D, S)) return VA_ERR_WORKSPACE;
    if (S > 1 && (long long)B * Hkv * ((R + rows - 1) / rows) > kCounters) return VA_ERR_TOO_LARGE;
    TreeParams p = {};
    p.K = static_cast<const uint8_t*>(b->K);
    p.V = static_cast<const uint8_t*>(b->V);
    p.scK = static_cast<const __half*>(b->scK);
    p.scV = static_cast<const __half*>(b->scV);
    p.q = static_cast<const __half*>(b->q);
    p.out = static_cast<__half*>(b->out);
    p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
    p.lens = lens;
    p.nodes = nodes;
    p.table = block_table;
    p.qs_b = qs[0];
    p.qs_t = qs[1];
    p.qs_h = qs[2];
    p.os_b = os[0];
    p.os_t = os[1];
    p.os_h = os[2];
    p.B = B;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.Q = Q;
    p.R = R;
    p.tiles = (R + rows - 1) / rows;
    p.S = S;
    p.max_pages = max_pages;
    p.page_rows = page_rows;
    p.num_pages = num_pages;
    divisor(page_rows, p.page_mul, p.page_shift);
    divisor(p.G, p.g_mul, p.g_shift);
    uint8_t* w = static_cast<uint8_t*>(ws);
    p.counters = reinterpret_cast<unsigned*>(w);
    w += kCounterBytes;
    p.ws_ml = reinterpret_cast<float*>(w);
    p.ws_o = reinterpret_cast<float*>(w + round256((size_t)B * Hq * Q * S * 8));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return D == 128 ? launch_tree_d128(fmt, p, rows, st) : launch_tree_d64(fmt, p, rows, st);
}

int va_append_packed(int fmt, const void* k, const void* v, int in_type, const long long* k_strides,
                     const long long* v_strides, const va_bufs* b, const int* block_table, int max_pages,
                     const int* cu_tokens, const int* pos, int T, int B, int Hkv, int page_rows, int num_pages, int D,
                     void* stream) {
    int rc = check_pool(fmt, b, B, max_pages, Hkv, page_rows, num_pages, D);
    if (rc) return rc;
    if (in_type < VA_FP32 || in_type > VA_BF16 || T < 0) return VA_ERR_INVALID;
    if (!block_table || !cu_tokens || !pos || (T > 0 && (!k || !v))) return VA_ERR_INVALID;
    if (!aligned16(k) || !aligned16(v) || !all_aligned4({block_table, cu_tokens, pos})) return VA_ERR_ALIGN;
    const long long dense[2] = {(long long)Hkv * D, D};
    const long long* ks = k_strides ? k_strides : dense;
    const long long* vs = v_strides ? v_strides : dense;
    const int step = in_type == VA_FP32 ? 4 : 8;  // 16-byte loads
    for (int i = 0; i < 2; ++i)
        if (ks[i] % step || vs[i] % step) return VA_ERR_ALIGN;
    if (T == 0) return VA_OK;
    AppendParams p = {};
    p.k = k;
    p.v = v;
    p.kt = ks[0];
    p.kh = ks[1];
    p.vt = vs[0];
    p.vh = vs[1];
    const PoolView pool = make_pool(fmt, b, Hkv, page_rows, num_pages, D, 1);
    p.K = pool.base[0];
    p.V = pool.base[1];
    p.scK = reinterpret_cast<__half*>(pool.base[2]);
    p.scV = reinterpret_cast<__half*>(pool.base[3]);
    p.table = block_table;
    p.cu = cu_tokens;
    p.pos = pos;
    p.T = T;
    p.B = B;
    p.Hkv = Hkv;
    p.D = D;
    p.max_pages = max_pages;
    p.page_rows = page_rows;
    p.num_pages = num_pages;
    divisor(page_rows, p.page_mul, p.page_shift);
    return launch_append_packed(fmt, in_type, p, static_cast<cudaStream_t>(stream));
}

int va_accept_tree(int fmt, const va_bufs* b, const int* block_table, int max_pages, const int* lens, const int* nodes,
                   const int* path, const int* accepted, int* new_lens, int B, int P, int Hkv, int page_rows,
                   int num_pages, int D, int layers, void* stream) {
    int rc = check_pool(fmt, b, B, max_pages, Hkv, page_rows, num_pages, D);
    if (!rc) rc = check_layers(Hkv, page_rows, num_pages, layers);
    if (rc) return rc;
    if (!block_table || !lens || !nodes || !path || !accepted || !new_lens || P < 1) return VA_ERR_INVALID;
    if (P > kAcceptMax || B > 65535) return VA_ERR_TOO_LARGE;
    if (!all_aligned4({block_table, lens, nodes, path, accepted, new_lens})) return VA_ERR_ALIGN;
    // (one CTA of a sequence writes its new length while the others still read)
    if (outputs_overlap({{new_lens, B}, {block_table, (long long)B * max_pages}, {lens, B}, {nodes, B}, {path, (long long)B * P}, {accepted, B}}, 1))
        return VA_ERR_INVALID;
    const PoolView pool = make_pool(fmt, b, Hkv, page_rows, num_pages, D, layers);
    AcceptParams p = {};
    p.K = pool.base[0];
    p.V = pool.base[1];
    p.scK = pool.base[2];
    p.scV = pool.base[3];
    p.table = block_table;
    p.lens = lens;
    p.nodes = nodes;
    p.path = path;
    p.accepted = accepted;
    p.new_lens = new_lens;
    p.layer_rows = (long long)num_pages * Hkv * page_rows;
    p.P = P;
    p.Hkv = Hkv;
    p.max_pages = max_pages;
    p.page_rows = page_rows;
    p.num_pages = num_pages;
    p.rb = pool.row_bytes[0];
    p.sb = has_scales(fmt) ? pool.row_bytes[2] : 0;
    return launch_accept_tree(p, B, layers, static_cast<cudaStream_t>(stream));
}

size_t va_pages_workspace_bytes(int B, int max_pages, int num_pages) {
    if (B < 1 || max_pages < 1 || num_pages < 1) return 0;
    // a fork: at most num_pages pages are given out, and three lists of sequences; a
    // compaction: the map and two lists of pages
    const size_t fork = (size_t)num_pages + 3 * (size_t)B, compact = 3 * (size_t)num_pages + 1;
    return round256(sizeof(int) * std::max(fork, compact));
}

int va_fork_pages(int fmt, const va_bufs* b, const int* refs, const int* block_table, const int* lens,
                  const int* parent, int* new_refs, int* new_table, int* new_lens, int* shortage, int Bin, int Bout,
                  int max_pages, int reserve, int Hkv, int page_rows, int num_pages, int D, int layers, void* ws,
                  size_t ws_bytes, void* stream) {
    int rc = check_pool(fmt, b, std::max(Bin, Bout), max_pages, Hkv, page_rows, num_pages, D);
    if (!rc) rc = check_layers(Hkv, page_rows, num_pages, layers);
    if (rc) return rc;
    if (page_rows % 8) return VA_ERR_UNSUPPORTED;
    if (Bin < 1 || Bout < 1 || reserve < 0) return VA_ERR_INVALID;
    if (!refs || !block_table || !lens || !parent || !new_refs || !new_table || !new_lens || !shortage) return VA_ERR_INVALID;
    if (Bin > kMaxForks || Bout > kMaxForks) return VA_ERR_TOO_LARGE;
    if (!all_aligned4({refs, block_table, lens, parent, new_refs, new_table, new_lens, shortage})) return VA_ERR_ALIGN;
    const Span outs[4] = {{new_refs, num_pages}, {new_table, (long long)Bout * max_pages}, {new_lens, Bout}, {shortage, 1}};
    const Span ins[4] = {{refs, num_pages}, {block_table, (long long)Bin * max_pages}, {lens, Bin}, {parent, Bout}};
    if (outputs_overlap({outs[0], outs[1], outs[2], outs[3], ins[0], ins[1], ins[2], ins[3]}, 4)) return VA_ERR_INVALID;
    if (!ws || !aligned_to(ws, 4) || ws_bytes < va_pages_workspace_bytes(Bout, max_pages, num_pages)) return VA_ERR_WORKSPACE;
    const Span scratch = {static_cast<int*>(ws), (long long)num_pages + 3ll * Bout};
    if (outputs_overlap({scratch, outs[0], outs[1], outs[2], outs[3], ins[0], ins[1], ins[2], ins[3]}, 1)) return VA_ERR_INVALID;
    ForkParams p = {};
    p.pool = make_pool(fmt, b, Hkv, page_rows, num_pages, D, layers);
    p.refs = refs;
    p.table = block_table;
    p.lens = lens;
    p.parent = parent;
    p.new_refs = new_refs;
    p.new_table = new_table;
    p.new_lens = new_lens;
    p.shortage = shortage;
    p.copy = static_cast<int*>(ws);
    p.free_list = p.copy + 3 * (size_t)Bout;
    p.Bin = Bin;
    p.Bout = Bout;
    p.max_pages = max_pages;
    p.reserve = reserve;
    return launch_fork_pages(p, static_cast<cudaStream_t>(stream));
}

int va_compact_pages(int fmt, const va_bufs* b, const int* refs, const int* block_table, int* new_refs, int* new_table,
                     int* used, int B, int max_pages, int Hkv, int page_rows, int num_pages, int D, int layers,
                     void* ws, size_t ws_bytes, void* stream) {
    int rc = check_pool(fmt, b, B, max_pages, Hkv, page_rows, num_pages, D);
    if (!rc) rc = check_layers(Hkv, page_rows, num_pages, layers);
    if (rc) return rc;
    if (page_rows % 8) return VA_ERR_UNSUPPORTED;
    if (!refs || !block_table || !new_refs || !new_table || !used) return VA_ERR_INVALID;
    if (!all_aligned4({refs, block_table, new_refs, new_table, used})) return VA_ERR_ALIGN;
    const long long entries = (long long)B * max_pages;
    const Span outs[3] = {{new_refs, num_pages}, {new_table, entries}, {used, 1}};
    const Span ins[2] = {{refs, num_pages}, {block_table, entries}};
    if (outputs_overlap({outs[0], outs[1], outs[2], ins[0], ins[1]}, 3)) return VA_ERR_INVALID;
    if (!ws || !aligned_to(ws, 4) || ws_bytes < va_pages_workspace_bytes(B, max_pages, num_pages)) return VA_ERR_WORKSPACE;
    if (outputs_overlap({{static_cast<int*>(ws), 3ll * num_pages + 1}, outs[0], outs[1], outs[2], ins[0], ins[1]}, 1)) return VA_ERR_INVALID;
    CompactParams p = {};
    p.pool = make_pool(fmt, b, Hkv, page_rows, num_pages, D, layers);
    p.refs = refs;
    p.table = block_table;
    p.new_refs = new_refs;
    p.new_table = new_table;
    p.used = used;
    p.count = static_cast<int*>(ws);
    p.map = p.count + 1;
    p.from = p.map + num_pages;
    p.to = p.from + num_pages;
    p.entries = entries;
    return launch_compact_pages(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
