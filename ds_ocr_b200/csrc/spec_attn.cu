// spec_attn.cu — attention of a tree of drafted tokens over the KV cache
// (ds_cuda_tree_attention_dev), and the trees' mask words.
//
// The R = n_nodes * group query rows that share a key head are taken
// together, in tiles of 8, 16, 128 or 256, so K and V are read once for all
// rows of a tile. The keys of a (sequence, key head, row tile) item come in
// tiles of 64: first the cached rows, then the tree's nodes. One pass keeps
// each row's running maximum, sum and weighted V in F32. All items' tiles form
// one list, cut into equal runs, one per persistent CTA: a ragged batch and a
// single long sequence are spread alike, and nothing about the lengths is
// needed on the host. A run that covers an item writes its result; an item cut
// between CTAs leaves (max, sum, weighted V) parts in the workspace, joined by
// sa_join_kernel. Small calls have a cluster per item instead, which joins its
// parts through its shared memory. The order of all sums is fixed by the
// lengths and the GPU's SM count, so results are repeatable.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "ctx.h"
#include "tmap.h"
#include "umma.cuh"

namespace ds {

constexpr int SA_MAX_NODES = 256;
constexpr int SA_MAX_KV = INT32_MAX - 1023;  // lengths are rounded up to whole tiles, and the nodes' tiles further, in 32 bits
constexpr int SA_THREADS = 128;
constexpr int SA_WARPS = SA_THREADS / 32;
constexpr int SA_CLUSTER = 16;  // CTAs of a cluster, at most
constexpr int SA_KT = 64;       // keys of a tile

struct SaArgs {
    ds_cuda_tree_attention_t d;
    int words;      // mask words per node
    int group;      // query heads per key head
    int rows;       // n_nodes * group
    int row_tiles;  // ceil(rows / row tile)
    int per_seq;    // n_kv_heads * row_tiles: items of a sequence
    int sms, ctas;  // SMs; runs the tile list is cut into, at most
    int cluster;    // CTAs of an item's cluster; 0: the list
    float scale2;   // scale * log2(e)
    unsigned *err;  // bounded waits that gave up
    float *part;    // workspace: [ctas][2][row tile][head_dim], then ...
    float2 *ml;     // ... [ctas][2][row tile] (max in log2 units, sum)
};

// ---- the tile list ---------------------------------------------------------
struct SaSeq {
    int len, cnt, cache_tiles, tiles;
};
template <int KT>
__device__ __forceinline__ SaSeq sa_seq(const ds_cuda_tree_attention_t &d, int b) {
    SaSeq s;
    const int len = d.lens[b];  // (beside the other load, not after it)
    s.cnt = d.nodes ? min(max(d.nodes[b], 0), d.n_nodes) : d.n_nodes;
    s.len = s.cnt ? min(max(len, 0), d.kv_max) : 0;  // no rows: one empty tile, whose results are zeros
    s.cache_tiles = (s.len + KT - 1) / KT;
    s.tiles = max(1, s.cache_tiles + (s.cnt + KT - 1) / KT);
    return s;
}
// Sums the sequences' tiles over the batch: returns the total, *mine the
// tiles before this thread's run of sequences [b0, b1), whose first is `own`.
// (The host refuses what could pass 2^31 tiles.)
template <int KT, int THREADS>
__device__ __forceinline__ int sa_scan(const SaArgs &a, int b0, int b1, const SaSeq &own, int *sh, int *mine) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = b0 < b1 ? own.tiles * a.per_seq : 0;
    for (int b = b0 + 1; b < b1; b++) s += sa_seq<KT>(a.d, b).tiles * a.per_seq;
    int v = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(DS_FULL, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    *mine = before + v - s;
    return total;
}
// The list cut into `ctas` runs whose lengths differ by one at most, the
// longer ones first.
struct SaCut {
    int ctas, len, more;
    __device__ __forceinline__ SaCut(int total, int most) {
        ctas = min(most, total);
        len = total / ctas;
        more = total - len * ctas;
    }
    __device__ __forceinline__ int start(int c) const { return c * len + min(c, more); }
    __device__ __forceinline__ int cta_of(int x) const {
        const int head = more * (len + 1);
        return x < head ? x / (len + 1) : more + (x - head) / len;
    }
};

// ---- loads and matrix instructions -----------------------------------------
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 block of 16-bit values, two a thread, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <bool F16> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
// Two values as three BF16 planes each: 24 bits, the value itself.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
    for (int k = 0; k < 3; k++) {
        p[k] = pack2<false>(x, y);
        x = __fsub_rn(x, __uint_as_float(p[k] << 16));
        y = __fsub_rn(y, __uint_as_float(p[k] & 0xffff0000u));
    }
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// With 16-bit queries the softmax weights are rounded to that type for the
// product with V (as V itself has been), while their sums stay in F32. FP16 ends
// at 2^-24: against a maximum of 1, weights below 2^-25 would be zero in the
// product, all of a result whose larger weights meet small V. Its weights are
// therefore 2^SA_LIFT times as large (maximum, sum and weighted V alike, so that
// nothing has to be taken back), which leaves an error of 2^-32 each. More would
// not fit: sums of weights may reach 2^15, and near 2^24 the maximum less
// SA_LIFT is rounded. (Where V is large throughout, the F32 sums end at 2^-25.)
constexpr float SA_LIFT = 7.f;
template <bool F16> __device__ __forceinline__ float sa_lift() { return F16 ? SA_LIFT : 0.f; }
// Byte offset of 16-byte chunk c of row r in a [rows][HD] 16-bit tile: the
// chunk is xor-ed with the row, so that ldmatrix's 8 rows meet 8 bank groups.
template <int HD> __device__ __forceinline__ uint32_t sw(int r, int c) { return (uint32_t)(r * HD * 2 + ((c ^ (r & 7)) << 4)); }

// Result or part of one row's dimensions [x, x + 4).
__device__ __forceinline__ void sa_store4(const ds_cuda_tree_attention_t &d, int64_t o, const float (&v)[4]) {
    if (d.type == DS_CUDA_SPEC_F32)
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(d.out) + o) = make_float4(v[0], v[1], v[2], v[3]);
    else if (d.type == DS_CUDA_SPEC_F16)
        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(d.out) + o) =
            make_uint2(pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3]));
    else
        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(d.out) + o) =
            make_uint2(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]));
}

// A part (weighted V u, sum l, factor f) added to (v, ll).
__device__ __forceinline__ void sa_add(float (&v)[4], float &ll, float4 u, float l, float f) {
    ll += l * f;
    v[0] += u.x * f;
    v[1] += u.y * f;
    v[2] += u.z * f;
    v[3] += u.w * f;
}
// Dimensions [c, c + 4) of a row's result, from its maximum, sum and weighted V.
__device__ __forceinline__ void sa_finish(const SaArgs &a, int b, int g, int row, int cnt, int c, float m, float l,
                                          float (&v)[4]) {
    const ds_cuda_tree_attention_t &d = a.d;
    const int nd = row / a.group, head = g * a.group + row % a.group;
    const bool none = nd >= cnt || l == 0.f;
    const float inv = 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = none ? 0.f : v[k] * inv;
    sa_store4(d, b * d.out_stride[0] + nd * d.out_stride[1] + head * d.out_stride[2] + c, v);
    if (d.lse && c == 0)
        d.lse[((size_t)b * d.n_nodes + nd) * d.n_heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.69314718f;
}

// ---- clusters ----------------------------------------------------------------
__device__ __forceinline__ int cluster_rank() {
    int r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int cluster_ctas() {
    int r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// CTA k's copy of a shared variable.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, int k) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(k));
    return r;
}
__device__ __forceinline__ float2 cluster_ld2(const float2 *p, int k) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(p, k)) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_ld4(const float4 *p, int k) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(p, k)) : "memory");
    return v;
}

// ---- a CTA's run of the list -------------------------------------------------
struct SaCursor {
    int b, g, rt, t;  // sequence, key head, row tile, tile of the item
    SaSeq s;
};
// The run's first tile and length. CLUSTER: an item is shared by one cluster,
// its tiles cut into the CTAs' runs. False: nothing to do (list only).
template <int KT, bool CLUSTER, int THREADS = SA_THREADS>
__device__ __forceinline__ bool sa_begin(const SaArgs &a, SaCursor &c, int &tiles) {
    __shared__ int sh_scan[THREADS / 32], sh_off, sh_b;
    __shared__ SaSeq sh_s;
    const int tid = threadIdx.x;
    if (CLUSTER) {
        const int rank = cluster_rank();
        c.b = blockIdx.z;
        c.g = blockIdx.y;
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(c.rt));
        c.s = sa_seq<KT>(a.d, c.b);
        const SaCut cut(c.s.tiles, cluster_ctas());
        c.t = rank < cut.ctas ? cut.start(rank) : 0;
        tiles = rank < cut.ctas ? cut.start(rank + 1) - c.t : 0;
        return true;
    }
    pdl_launch();
    const int chunk = (a.d.batch + THREADS - 1) / THREADS;
    const int b0 = min(a.d.batch, tid * chunk), b1 = min(a.d.batch, b0 + chunk);
    int at;
    SaSeq s = sa_seq<KT>(a.d, min(b0, a.d.batch - 1));
    const int total = sa_scan<KT, THREADS>(a, b0, b1, s, sh_scan, &at);
    const SaCut cut(total, a.ctas);
    if ((int)blockIdx.x >= cut.ctas) return false;
    const int first = cut.start(blockIdx.x);
    tiles = cut.start(blockIdx.x + 1) - first;
    for (int b = b0; b < b1; b++) {
        if (b > b0) s = sa_seq<KT>(a.d, b);
        const int n = s.tiles * a.per_seq;
        if (at <= first && first < at + n) {
            sh_b = b;
            sh_s = s;
            sh_off = first - at;
        }
        at += n;
    }
    __syncthreads();
    c.b = sh_b;
    c.s = sh_s;
    const int off = sh_off / c.s.tiles;
    c.t = sh_off - off * c.s.tiles;
    c.rt = off % a.row_tiles;
    c.g = off / a.row_tiles;
    return true;
}
template <int KT> __device__ __forceinline__ void sa_next(const SaArgs &a, SaCursor &c) {
    if (++c.t < c.s.tiles) return;
    c.t = 0;
    if (++c.rt < a.row_tiles) return;
    c.rt = 0;
    if (++c.g < a.d.n_kv_heads) return;
    c.g = 0;
    if (++c.b < a.d.batch) c.s = sa_seq<KT>(a.d, c.b);
}
// Where a tile's rows are: K and V planes, row strides, the valid rows (may
// be none or more than the tile's).
struct SaTile {
    bool node;
    int r0, valid;
    const uint16_t *base[2][2];
    int64_t step[2];
    bool lo[2];
};
template <int KT> __device__ __forceinline__ SaTile sa_tile(const ds_cuda_tree_attention_t &d, const SaCursor &c) {
    SaTile s;
    s.node = c.t >= c.s.cache_tiles;
    s.r0 = (s.node ? c.t - c.s.cache_tiles : c.t) * KT;
    s.valid = (s.node ? c.s.cnt : c.s.len) - s.r0;
    const int64_t *ks = s.node ? d.tree_k_stride : d.k_stride, *vs = s.node ? d.tree_v_stride : d.v_stride;
    const int64_t ko = c.b * ks[0] + c.g * ks[1] + (int64_t)s.r0 * ks[2], vo = c.b * vs[0] + c.g * vs[1] + (int64_t)s.r0 * vs[2];
    const void *k_lo = s.node ? d.tree_k_lo : d.k_lo, *v_lo = s.node ? d.tree_v_lo : d.v_lo;
    s.base[0][0] = (const uint16_t *)(s.node ? d.tree_k : d.k) + ko;
    s.base[0][1] = (const uint16_t *)k_lo + ko;
    s.base[1][0] = (const uint16_t *)(s.node ? d.tree_v : d.v) + vo;
    s.base[1][1] = (const uint16_t *)v_lo + vo;
    s.step[0] = ks[2];
    s.step[1] = vs[2];
    s.lo[0] = k_lo != nullptr;
    s.lo[1] = v_lo != nullptr;
    return s;
}
// Dimension c of row r of a part in shared memory is at c ^ sa_swz(r).
__device__ __forceinline__ int sa_swz(int r) { return ((r >> 1) & 3) << 3; }
// A CTA's part of an item, from KS warps' parts of each row: given to
// put(row, c, max, sum, values of dimensions [c, c + 4)).
template <int RT, int HD, int KS, class ML, class PART, class PUT>
__device__ __forceinline__ void sa_merge(ML ml_of, PART part_of, PUT put) {
    for (int x = threadIdx.x; x < RT * (HD / 4); x += SA_THREADS) {
        const int r = x / (HD / 4), c = 4 * (x % (HD / 4));
        float mm = -__FLT_MAX__, ll = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KS; w++) mm = fmaxf(mm, ml_of(w, r).x);
#pragma unroll
        for (int w = 0; w < KS; w++) {
            const float2 ml = ml_of(w, r);
            sa_add(v, ll, *reinterpret_cast<const float4 *>(part_of(w, r, c)), ml.y, ex2(ml.x - mm));
        }
        put(r, c, mm, ll, v);
    }
}
// What a CTA does with its part of an item: keep it for the cluster, write
// the result, or leave it in the workspace (slot 0: a run's first item,
// begun by an earlier CTA; 1: its last).
template <int RT, int HD, bool CLUSTER>
__device__ __forceinline__ void sa_put(const SaArgs &a, const SaCursor &c, bool first, bool last, float4 *sh_part,
                                       float2 *sh_pml, int r, int col, float m, float l, float (&v)[4]) {
    const int row = c.rt * RT + r;
    if (row >= a.rows) return;
    if (CLUSTER) {
        sh_part[r * (HD / 4) + col / 4] = make_float4(v[0], v[1], v[2], v[3]);
        if (col == 0) sh_pml[r] = make_float2(m, l);
    } else if (first && last) {
        sa_finish(a, c.b, c.g, row, c.s.cnt, col, m, l, v);
    } else {
        const size_t pr = ((size_t)blockIdx.x * 2 + first) * RT + r;
        *reinterpret_cast<float4 *>(a.part + pr * HD + col) = make_float4(v[0], v[1], v[2], v[3]);
        if (col == 0) a.ml[pr] = make_float2(m, l);
    }
}
// The cluster's parts joined, each CTA a share of the rows and dimensions.
template <int RT, int HD>
__device__ __forceinline__ void sa_cluster_join(const SaArgs &a, const SaCursor &c, const float4 *sh_part,
                                                const float2 *sh_pml) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // every CTA's part is in its shared memory
    const int used = min(cluster_ctas(), c.s.tiles), left = min(RT, a.rows - c.rt * RT);
    static_assert(RT * (HD / 4) <= 8 * SA_THREADS, "a cluster's threads take four dimensions of a row at most");
    const int x = cluster_rank() * SA_THREADS + threadIdx.x, r = x / (HD / 4);
    const bool mine = x < left * (HD / 4);
    float mm = -__FLT_MAX__, ll = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
        // (loads in batches: one after the other they take 3000 cycles)
        float2 ml[SA_CLUSTER];
#pragma unroll
        for (int k = 0; k < SA_CLUSTER; k++) ml[k] = cluster_ld2(&sh_pml[r], min(k, used - 1));
#pragma unroll
        for (int k = 0; k < SA_CLUSTER; k++) mm = fmaxf(mm, ml[k].x);
#pragma unroll
        for (int k0 = 0; k0 < SA_CLUSTER; k0 += 8) {
            if (k0 >= used) break;
            float4 u[8];
#pragma unroll
            for (int k = 0; k < 8; k++) u[k] = cluster_ld4(&sh_part[x], min(k0 + k, used - 1));
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k0 + k < used) sa_add(v, ll, u[k], ml[k0 + k].y, ex2(ml[k0 + k].x - mm));
        }
    }
    __syncwarp();
    cluster_arrive();  // before the results are written: it would wait for them
    if (mine) sa_finish(a, c.b, c.g, c.rt * RT + r, c.s.cnt, 4 * (x % (HD / 4)), mm, ll, v);
    cluster_wait();  // no CTA leaves while another reads its part
}

// ---- few rows: up to 16 at a time ------------------------------------------------
// Keys take the 16-row side of the matrix instructions and the query rows the
// 8-column side (S^T = K Q^T, O^T = V^T P^T), so up to 8 rows waste nothing and
// K and V fragments serve all rows. A tile is 64 keys, 16 per warp; a warp
// loads, multiplies and sums its own keys, with no barrier but at an item's
// end. Its K and V rows of a tile are a unit each in a ring of three: while
// one is used, two are in flight, with eight warps an SM 128 KB of them. The
// queries stay in registers. F32 queries and weights are three BF16 planes
// (exact), K and V two; products below 2^-24 of the largest are left out.
// (Times here and below are of calls in a graph, the same inputs each time.)
// Bound by the memory for 8 rows: 64 streams of 10 heads, up to 1325 tokens, F32
// in two planes, 93 us, 6.0 TB/s. Two groups of F32 rows take 126 us for them:
// five products an element with eight warps an SM, short of both the memory's
// rate and mma.sync's (a quarter of it). More rows read K and V once per 16:
// 243 us for 32, 480 us for 64 nodes. One stream of 662 tokens is bound by
// latency: lengths, one tile's rows, the tile's steps, the cluster's join follow
// one another: 7.2 us for one node, 9.1 us for 16.
template <int HD_, int NG_, int PL_, int QT_> struct SaFew {
    static constexpr int HD = HD_, NG = NG_, PL = PL_, QT = QT_;
    static constexpr int QP = QT == DS_CUDA_SPEC_F32 ? 3 : 1;
    static constexpr int RT = 8 * NG, KT = SA_KT;
    static constexpr int PLANE = 16 * HD * 2, UNIT = PL * PLANE;  // of a warp
    static constexpr int SMEM = SA_WARPS * 3 * UNIT;
    static constexpr int PHASES = RT * HD * 4 > UNIT ? RT * HD * 4 / UNIT : 1;  // of a join through one unit a warp
    static constexpr int FIT = (226 << 10) / (SMEM + 3072);
    static constexpr int MOST = HD == 128 && QP == 3 && NG == 2 ? 2 : HD == 128 || QP == 3 ? 3 : 4;  // by registers
    static constexpr int PER_SM = FIT < MOST ? FIT : MOST;
    static_assert(RT * HD * 4 <= 2 * UNIT, "a CTA's part takes two units at most");
};

template <class S, bool CLUSTER>
__global__ void __launch_bounds__(SA_THREADS, S::PER_SM) sa_few_kernel(const __grid_constant__ SaArgs a) {
    constexpr int HD = S::HD, NG = S::NG, CH = HD / 8, KK = HD / 16, NL = NG == 1 ? 4 : 2;
    constexpr int RS = 32 / CH;  // rows a warp's 16-byte lanes cover at once
    constexpr bool F16 = S::QT == DS_CUDA_SPEC_F16, F32 = S::QT == DS_CUDA_SPEC_F32;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float2 sh_ml[SA_WARPS][S::RT], sh_pml[S::RT];
    // a cluster's part: over the first warp's last unit and the second's first
    float4 *const sh_part = reinterpret_cast<float4 *>(smem + 2 * S::UNIT);
    const ds_cuda_tree_attention_t &d = a.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, gc = lane & 3;
    SaCursor ld;
    int tiles;
    if (!sa_begin<S::KT, CLUSTER>(a, ld, tiles)) return;
    SaCursor cu = ld;
    const SaCursor item = ld;  // CLUSTER's one item
    uint8_t *const mine = smem + warp * 3 * S::UNIT;
    auto wrap = [](int x) { return x >= 3 ? x - 3 : x; };

    // Loads: this warp's 16 rows of the cursor's tile, K or V. The pointers
    // (of this lane's first row and 16 bytes) step from tile to tile and are
    // set anew where an item or its tree begins.
    const int cc = lane % CH, rr = lane / CH;
    const uint16_t *from[2][2];
    int64_t step[2];
    bool lo[2];
    int left = 0;  // valid rows from this warp's first on
    auto aim = [&]() {
        const SaTile src = sa_tile<S::KT>(d, ld);
        left = src.valid - 16 * warp;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            step[kv] = src.step[kv] * RS;
            lo[kv] = src.lo[kv];
#pragma unroll
            for (int p = 0; p < S::PL; p++) from[kv][p] = src.base[kv][p] + (16 * warp + rr) * src.step[kv] + 8 * cc;
        }
    };
    auto load = [&](int kv, int slot) {
        const uint32_t dst = smem_u32(mine) + slot * S::UNIT;
        if (left >= 16 && (S::PL == 1 || lo[kv])) {
#pragma unroll
            for (int p = 0; p < S::PL; p++) {
                const uint16_t *x = from[kv][p];
#pragma unroll
                for (int r = 0; r < 16; r += RS, x += step[kv]) cp16(dst + p * S::PLANE + sw<HD>(rr + r, cc), x);
            }
        } else if (left > 0) {  // rows past the valid ones are zeros, and so is a plane that is not there
#pragma unroll
            for (int p = 0; p < S::PL; p++) {
                const uint16_t *x = from[kv][p];
#pragma unroll
                for (int r = 0; r < 16; r += RS, x += step[kv]) {
                    const bool ok = rr + r < left && (p == 0 || lo[kv]);
                    cp16(dst + p * S::PLANE + sw<HD>(rr + r, cc), ok ? x : d.q, ok);
                }
            }
        }
        cp_commit();
    };
    auto advance = [&]() {
        const int was = ld.t;
        const bool tree = was + 1 == ld.s.cache_tiles;
        sa_next<S::KT>(a, ld);
        if (ld.t == 0 || tree || was >= ld.s.cache_tiles) {
            if (ld.b < d.batch) aim();
            return;
        }
        left -= S::KT;
#pragma unroll
        for (int kv = 0; kv < 2; kv++)
#pragma unroll
            for (int p = 0; p < S::PL; p++) from[kv][p] += step[kv] * (S::KT / RS);
    };
    uint64_t bits[NG][2];                 // of rows 2 gc and 2 gc + 1 of each group, for the tree's tile at hand
    auto word = [&](int n, int e, int k) -> uint64_t {
        const int row = cu.rt * S::RT + 8 * n + 2 * gc + e, nd = row / a.group, left = cu.s.cnt - 64 * k;
        if (row >= a.rows || nd >= cu.s.cnt || left <= 0) return 0;
        return d.mask[((size_t)cu.b * d.n_nodes + nd) * a.words + k] & (left < 64 ? (1ull << left) - 1 : ~0ull);
    };
    // an item's queries as they are (16-bit ones two in the first float)
    float2 qu[NG][KK][2];
    auto q_load = [&]() {
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const int row = cu.rt * S::RT + 8 * n + gr;
            const bool ok = row < a.rows;
            const int64_t qo = ok ? cu.b * d.q_stride[0] + (row / a.group) * d.q_stride[1] +
                                        (cu.g * a.group + row % a.group) * d.q_stride[2] + 2 * gc : 0;
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float2 &u = qu[n][kk][h];
                    u = make_float2(0.f, 0.f);
                    if (!ok) continue;
                    if (F32) u = *reinterpret_cast<const float2 *>((const float *)d.q + qo + 16 * kk + 8 * h);
                    else u.x = *reinterpret_cast<const float *>((const uint16_t *)d.q + qo + 16 * kk + 8 * h);
                }
#pragma unroll
            for (int e = 0; e < 2; e++) bits[n][e] = word(n, e, 0);
        }
    };
    // The first item's before the rows: they arrive while those are asked for.
    // Not where the registers are short (F32, 16 rows or three CTAs an SM): held
    // ahead they make the loop spill, 64 streams of 10 heads, up to 1325 tokens:
    // 16 / 32 / 64 nodes 182 / 348 / 700 us instead of 126 / 243 / 480, 8 nodes
    // on a single plane 61 instead of 54.
    constexpr bool AHEAD = !F32 || (NG == 1 && S::PL == 2);
    if (AHEAD) q_load();
    if (tiles > 0) {
        aim();
        load(0, 0);
        load(1, 1);
        advance();
    }

    uint32_t qf[NG][S::QP][KK][2];
    float o[KK][NG][4], m[NG][2], l[NG][2];
    bool fresh = true, whole = cu.t == 0;
    int slot = 0;  // of K; V's follows it, then the next tile's
    for (int i = 0; i < tiles; i++, slot = wrap(slot + 2)) {
        if (fresh) {
            fresh = false;
            if (!AHEAD || i > 0) q_load();
#pragma unroll
            for (int n = 0; n < NG; n++) {
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (F32) {
                            uint32_t p[3];
                            split3(qu[n][kk][h].x, qu[n][kk][h].y, p);
#pragma unroll
                            for (int k = 0; k < S::QP; k++) qf[n][k][kk][h] = p[k];
                        } else {
                            qf[n][0][kk][h] = __float_as_uint(qu[n][kk][h].x);
                        }
                    }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    m[n][e] = -__FLT_MAX__;
                    l[n][e] = 0.f;
                }
#pragma unroll
                for (int t = 0; t < KK; t++) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
            }
        }
        cp_wait<1>();
        __syncwarp();
        const bool more = i + 1 < tiles;
        if (more) load(0, wrap(slot + 2));
        else cp_commit();

        const bool node = cu.t >= cu.s.cache_tiles;
        const int tree = cu.t - cu.s.cache_tiles;
        const int valid = (node ? cu.s.cnt - tree * S::KT : cu.s.len - cu.t * S::KT) - 16 * warp;  // of this warp's keys
        if (tree > 0)  // (the first tile's came with the queries)
#pragma unroll
            for (int n = 0; n < NG; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) bits[n][e] = word(n, e, tree);
        uint32_t pf[NG][S::QP][2];
        if (valid > 0) {
            const uint32_t k_s = smem_u32(mine) + slot * S::UNIT;
            // scores of 16 keys and 8 NG rows; the planes' products of lower
            // orders apart (shorter chains, smaller rounding)
            float s[NG][4], low[F32 ? NG : 1][NL][4];
#pragma unroll
            for (int n = 0; n < NG; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[n][e] = 0.f;
                    if (F32)
#pragma unroll
                        for (int x = 0; x < NL; x++) low[n][x][e] = 0.f;
                }
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                uint32_t kf[S::PL][4];
#pragma unroll
                for (int p = 0; p < S::PL; p++) ldsm4(kf[p], k_s + p * S::PLANE + sw<HD>(lane & 15, 2 * kk + (lane >> 4)));
#pragma unroll
                for (int pk = 0; pk < S::PL; pk++)
#pragma unroll
                    for (int pq = 0; pq < S::QP; pq++)
                        if (pq + pk < 3)
#pragma unroll
                            for (int n = 0; n < NG; n++) {
                                const int x = NG == 1 ? (pq == 0 ? 0 : pq == 2 ? 3 : pk + 1) : pq + pk - 1;
                                mma16<F16>(pq + pk ? low[F32 ? n : 0][x & (NL - 1)] : s[n], kf[pk], qf[n][pq][kk][0], qf[n][pq][kk][1]);
                            }
            }
            if (F32)
#pragma unroll
                for (int n = 0; n < NG; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = low[n][0][e] + low[n][1][e];
                        if (NL == 4) x += low[n][2 & (NL - 1)][e] + low[n][3 & (NL - 1)][e];
                        s[n][e] += x;
                    }
            // element e: key gr + 8 (e >> 1), row 2 gc + (e & 1) of group n
            const bool masked = node || valid < 16;
            uint32_t see = ~0u;  // 4 bits per group
            if (masked) {
                see = 0;
#pragma unroll
                for (int n = 0; n < NG; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = gr + 8 * (e >> 1);
                        const bool ok = node ? (bits[n][e & 1] >> (16 * warp + key)) & 1 : key < valid;
                        see |= (uint32_t)ok << (4 * n + e);
                    }
            }
            float mx[NG][2];
            bool grew = false;
#pragma unroll
            for (int n = 0; n < NG; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    mx[n][e] = m[n][e];
                    if (see >> (4 * n + e) & 1) mx[n][e] = fmaxf(mx[n][e], __fmul_rn(s[n][e], a.scale2));
                    if (see >> (4 * n + e + 2) & 1) mx[n][e] = fmaxf(mx[n][e], __fmul_rn(s[n][e + 2], a.scale2));
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) mx[n][e] = fmaxf(mx[n][e], __shfl_xor_sync(DS_FULL, mx[n][e], w));
                    grew |= mx[n][e] > m[n][e];
                }
            }
            if (__any_sync(DS_FULL, grew)) {
#pragma unroll
                for (int n = 0; n < NG; n++) {
                    const float f0 = ex2(m[n][0] - mx[n][0]), f1 = ex2(m[n][1] - mx[n][1]);
                    m[n][0] = mx[n][0];
                    m[n][1] = mx[n][1];
                    l[n][0] *= f0;
                    l[n][1] *= f1;
#pragma unroll
                    for (int t = 0; t < KK; t++) {
                        o[t][n][0] *= f0;
                        o[t][n][1] *= f1;
                        o[t][n][2] *= f0;
                        o[t][n][3] *= f1;
                    }
                }
            }
            // the weights, and their fragments: the score fragment's 8 x 8
            // blocks [key][row] transposed are those of P^T [key] for the rows
            // (FP16: from the rounded products that the maximum was taken of,
            // so that the largest weight is 2^SA_LIFT whatever the scores' size)
#pragma unroll
            for (int n = 0; n < NG; n++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = F16 ? __fsub_rn(__fmul_rn(s[n][e], a.scale2), m[n][e & 1] - sa_lift<F16>())
                                        : __fmaf_rn(s[n][e], a.scale2, -m[n][e & 1]);
                    s[n][e] = see >> (4 * n + e) & 1 ? ex2(x) : 0.f;
                    l[n][e & 1] += s[n][e];
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t p[3];
                    if (F32) split3(s[n][2 * h], s[n][2 * h + 1], p);
                    else p[0] = pack2<F16>(s[n][2 * h], s[n][2 * h + 1]);
#pragma unroll
                    for (int k = 0; k < S::QP; k++) pf[n][k][h] = transpose8(p[k]);
                }
            }
        }
        cp_wait<1>();
        __syncwarp();
        if (more) {
            load(1, slot);
            advance();
        } else {
            cp_commit();
        }
        if (valid > 0) {
            uint8_t *const vs = mine + wrap(slot + 1) * S::UNIT;
            const uint32_t v_s = smem_u32(vs);
            if (node) {
                // A node's V may hold NaN or infinities that some rows must not
                // see, and 0 * NaN would spread through the product: such values
                // are added here to the rows that attend them, then zeroed.
                constexpr uint32_t E = F16 ? 0x7c007c00u : 0x7f807f80u;
                bool bad = false;
                for (int x = lane; x < S::UNIT / 16; x += 32) {
                    const uint4 u = reinterpret_cast<const uint4 *>(vs)[x];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t e = ((&u.x)[k] & E) ^ E;
                        bad |= !(e & 0xffffu) || !(e >> 16);
                    }
                }
                if (__any_sync(DS_FULL, bad)) {
                    for (int key = 0; key < 16; key++)
#pragma unroll
                        for (int t = 0; t < KK; t++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                float v = 0.f;
#pragma unroll
                                for (int p = 0; p < S::PL; p++) {
                                    const uint16_t w = *reinterpret_cast<const uint16_t *>(vs + p * S::PLANE + sw<HD>(key, 2 * t + h) + 2 * gr);
                                    v += F16 ? __half2float(__ushort_as_half(w)) : __uint_as_float((uint32_t)w << 16);
                                }
                                if (!isfinite(v))
#pragma unroll
                                    for (int n = 0; n < NG; n++)
#pragma unroll
                                        for (int e = 0; e < 2; e++)
                                            if (bits[n][e] >> (16 * warp + key) & 1) o[t][n][2 * h + e] += v;
                            }
                    __syncwarp();
                    for (int x = lane; x < 16 * HD; x += 32) {
                        const uint32_t off = sw<HD>(x / HD, x % HD / 8) + 2 * (x % 8);
                        bool nf = false;
#pragma unroll
                        for (int p = 0; p < S::PL; p++)
                            nf |= (*reinterpret_cast<uint16_t *>(vs + p * S::PLANE + off) & (E & 0xffff)) == (E & 0xffff);
                        if (nf)
#pragma unroll
                            for (int p = 0; p < S::PL; p++) *reinterpret_cast<uint16_t *>(vs + p * S::PLANE + off) = 0;
                    }
                    __syncwarp();
                }
            }
            // O^T += V^T P^T
#pragma unroll
            for (int t = 0; t < KK; t++) {
                uint32_t vf[S::PL][4];
#pragma unroll
                for (int p = 0; p < S::PL; p++)
                    ldsm4t(vf[p], v_s + p * S::PLANE + sw<HD>((lane & 7) + ((lane >> 4) << 3), 2 * t + ((lane >> 3) & 1)));
                // (F32: a tile's products apart, added with rounding to nearest:
                // the tensor cores' own sums round towards zero, which adds up
                // over a long cache)
                float x[F32 ? NG : 1][4] = {};
#pragma unroll
                for (int pk = S::PL - 1; pk >= 0; pk--)
#pragma unroll
                    for (int pq = S::QP - 1; pq >= 0; pq--)
                        if (pq + pk < 3)
#pragma unroll
                            for (int n = 0; n < NG; n++) mma16<F16>(F32 ? x[F32 ? n : 0] : o[t][n], vf[pk], pf[n][pq][0], pf[n][pq][1]);
                if (F32)
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[t][n][e] += x[F32 ? n : 0][e];
            }
        }

        const bool end = cu.t + 1 == cu.s.tiles;
        if (end || i + 1 == tiles) {
            // the item, or this CTA's part of it, is done: the warps' parts are
            // joined through V's units, which are free (a cluster's run ends
            // here, with every unit free: through the second ones), in phases
            // where they are smaller than a part
            constexpr int STEP = 3 * S::UNIT / 4, COLS = HD / S::PHASES;
            const int js = CLUSTER ? 1 : wrap(slot + 1);
            float *const so = reinterpret_cast<float *>(mine + js * S::UNIT);
            const float *const parts = reinterpret_cast<const float *>(smem + js * S::UNIT);
#pragma unroll
            for (int n = 0; n < NG; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(DS_FULL, l[n][e], w);
                    if (gr == 0) sh_ml[warp][8 * n + 2 * gc + e] = make_float2(m[n][e] - sa_lift<F16>(), l[n][e]);
                }
#pragma unroll
            for (int ph = 0; ph < S::PHASES; ph++) {
                // (a cluster's other units may still be read by slower warps)
                if (CLUSTER && ph == 0) __syncthreads();
                else __syncwarp();
#pragma unroll
                for (int n = 0; n < NG; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int t = 0; t < KK / S::PHASES; t++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const int r = 8 * n + 2 * gc + e;
                                so[r * COLS + ((16 * t + 8 * h + gr) ^ sa_swz(r))] = o[t + ph * (KK / S::PHASES)][n][2 * h + e];
                            }
                __syncthreads();
                sa_merge<S::RT, COLS, SA_WARPS>(
                    [&](int w, int r) { return sh_ml[w][r]; },
                    [&](int w, int r, int c) { return parts + w * STEP + r * COLS + (c ^ sa_swz(r)); },
                    [&](int r, int c, float mm, float ll, float (&v)[4]) {
                        sa_put<S::RT, HD, CLUSTER>(a, cu, whole, end, sh_part, sh_pml, r, c + ph * COLS, mm, ll, v);
                    });
                __syncthreads();  // the join's readers are done: the units may be refilled
            }
            fresh = true;
            whole = true;
        }
        sa_next<S::KT>(a, cu);
    }
    cp_wait<0>();
    if (CLUSTER) sa_cluster_join<S::RT, HD>(a, item, sh_part, sh_pml);
}

// ---- many rows: tcgen05 ----------------------------------------------------------
// 16-bit types with more than 16 rows. The 128 query rows of a block are the
// rows of tcgen05.mma (M = 128, accumulators in tensor memory); two softmax
// groups of 256 threads, two a row, work on two streams:
//   DUAL (more than 128 rows): the streams are two blocks of rows that share
//        every K and V tile;
//   else: one block of rows, the streams take the even and the odd tiles, and
//        their results are joined where they are written.
// Per stream and tile of 64 keys: S = Q K^T (both from shared memory) into one
// of two buffers in tensor memory; a thread reads half a row of S, takes
// 2^(S - m) and stores it, in the place of S, as P; O += P V with P as the A
// operand. A warp of its own issues a stream's products (issuing takes about
// 60 cycles a product, which one warp could not do for both), the next tile's
// S before this one's P is there. m is the row's maximum of its first tile,
// or of a later one whose weights passed 2^10 (FP16: 2^8), so that O is rarely
// rescaled. P has the cache's type: its rounding is of the same size as V's. Bound by
// the memory at 124 rows (8 streams, 32 heads on 8, head_dim 128, up to 8191
// tokens: 47.4 us, 3.9 TB/s over the whole call, the runs themselves at the
// memory's rate, 10 us of start and item ends, 8 us of join), by the softmax at
// 512 rows (one stream, 16 heads on 2, head_dim 64, 131071 tokens: 78 us, 440
// TFLOP/s; a step of 2 x 128 rows and 64 keys takes 1850 cycles, 1024 of them
// the exponentials' least, and a CTA's 56 steps 53 us; the rest is start, parts
// and join). Tried for the latter: P in columns of its own, which
// lets S be issued a product earlier (82 us), turns of the two streams (97
// against 85 us at the time), packed F32 operations (no change).
// Two producer warps bring K and V rows into a ring each (of K and of V, or of
// the streams) in the 128-byte swizzle, in the order the products take them.
constexpr int TC_SOFTMAX = 512, TC_PRODUCERS = 64, TC_THREADS = TC_SOFTMAX + TC_PRODUCERS + 64;
constexpr int TC_ALL = 9;  // barrier of the softmax threads (1 .. 8: of the two warps of 32 rows)
constexpr uint32_t TC_DHI = 64u | (1u << 14) | (2u << 29);  // descriptors' high word: 1024 B between 8-row atoms, 128-byte swizzle
template <int HD_, bool DUAL_, int QT_> struct SaMany {
    static constexpr int HD = HD_, QT = QT_, PL = 1;
    static constexpr bool DUAL = DUAL_;
    static constexpr int RT = DUAL ? 256 : 128;
    static constexpr int KT = SA_KT;
    static constexpr int SUB = KT * 128;           // 64 dimensions of a unit
    static constexpr int UNIT = KT * HD * 2;       // 16 KB, 8 KB for head_dim 64
    static constexpr int QSUB = 128 * 128, QBLOCK = QSUB * (HD / 64);
    static constexpr int UNITS = HD == 64 ? 16 : DUAL ? 8 : 10;
    static constexpr int RING = UNITS / 2;         // two rings: of K and of V (DUAL), or of the streams
    static constexpr int SMEM = RT / 128 * QBLOCK + UNITS * UNIT + 1024;
    static constexpr int PER_SM = 1;
    // tensor-memory columns: S (two buffers a stream, P in the first half of each), O
    static constexpr uint32_t TS = 0, TO = 4 * KT;
    static_assert(TO + 2 * HD <= 512, "tensor memory");
    // a stream's ring holds, of an item with n of its tiles, K of two tiles,
    // then V and K in turn. The place of K and V of tile t, and what is at a
    // place.
    static __device__ __forceinline__ int place_k(int t) { return t < 2 ? t : 2 * t - 1; }
    static __device__ __forceinline__ int place_v(int t, int n) { return min(2, n) + t + min(t, max(0, n - 2)); }
    static __device__ __forceinline__ int at(int place, int n, int &kv) {
        const int r = place - min(2, n), m = max(0, n - 2);
        kv = r >= 0 && (r >= 2 * m || !(r & 1));
        return r < 0 ? place : r >= 2 * m ? r - m : kv ? r / 2 : 2 + r / 2;
    }
};

__device__ __forceinline__ void mbar_arrive_n(uint64_t *bar, uint32_t n) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0], %1;" :: "r"(smem_u32(bar)), "r"(n) : "memory");
}
// A wait that gives up after two seconds: the failure is recorded in *err (if
// given) and everyone leaves.
__device__ __forceinline__ bool tc_wait(uint64_t *bar, uint32_t parity, unsigned *err) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = ds_gtime();
    do {
        for (int i = 0; i < 64; i++)
            if (mbar_try_wait(bar, parity)) return true;
    } while (ds_gtime() - t0 < 2000000000ull);
    if (err) atomicAdd(err, 1u);
    return false;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) :: "memory");
    return r != 0;
}
// tcgen05.mma with both operands in shared memory, the descriptors given as
// low words and a common high word.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t alo, uint32_t blo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .b64 ad, bd;\n\t.reg .pred p;\n\t"
        "mov.b64 ad, {%1, %3};\n\tmov.b64 bd, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %4, p;\n\t}"
        :: "r"(d), "r"(alo), "r"(blo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void cp_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(n) : "memory"); }
// ... returning whether any of them passed `x`.
__device__ __forceinline__ bool bar_or(int id, int n, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)x), "r"(id), "r"(n) : "memory");
    return r != 0;
}
// ... whether all of them passed `ok`.
__device__ __forceinline__ bool bar_and(int id, int n, bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)ok), "r"(id), "r"(n) : "memory");
    return r != 0;
}

// Tensor maps of the cache's K and V (64-dimension boxes of KT rows): whole
// tiles are one thread's TMA loads, where the strides allow a map; partial
// ones and the nodes' are copied with zeros past their rows.
struct SaManyArgs {
    CUtensorMap map[2];
    SaArgs a;
    int mapped;
    int dim[2][3];  // the map's dimension (1, 2, 3) of row, head, sequence
};
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;"
        :: "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// Queries and mask words into L2 (a share of a CTA each) before K's and V's
// loads fill the queues to the memory: behind them they take 3 us.
template <int HD> __device__ __forceinline__ void sa_warm(const SaArgs &a) {
    const ds_cuda_tree_attention_t &d = a.d;
    constexpr int LINES = HD * 2 / 128;
    const int most = 2 * gridDim.x * TC_THREADS, step = gridDim.x * TC_THREADS, x0 = blockIdx.x * TC_THREADS + threadIdx.x;
    const int64_t rows = (int64_t)d.batch * d.n_nodes, bytes = rows * a.words * 8, lines = rows * d.n_heads * LINES;
    for (int x = x0; x < most && x < lines; x += step) {
        const int r = x / LINES, nd = r / d.n_heads;
        const uint16_t *const q = (const uint16_t *)d.q + nd / d.n_nodes * d.q_stride[0] + nd % d.n_nodes * d.q_stride[1] +
                                  r % d.n_heads * d.q_stride[2] + x % LINES * 64;
        asm volatile("prefetch.global.L2 [%0];" :: "l"(q));
    }
    for (int64_t x = (int64_t)x0 * 128; x < bytes; x += (int64_t)step * 128)
        asm volatile("prefetch.global.L2 [%0];" :: "l"(reinterpret_cast<const char *>(d.mask) + x));
}

template <class S>
__global__ void __launch_bounds__(TC_THREADS, 1) sa_many_kernel(const __grid_constant__ SaManyArgs args) {
    const SaArgs &a = args.a;
    constexpr int HD = S::HD, KT = S::KT, CH = HD / 8, NU = S::UNITS, STEP = S::DUAL ? 1 : 2;
    constexpr bool F16 = S::QT == DS_CUDA_SPEC_F16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *const ring = smem + S::RT / 128 * S::QBLOCK;
    __shared__ uint64_t full[NU], empty[NU], qfull, sfull[2][2], pfull[2][2], pvdone[2], odone[2], drain[2];
    __shared__ uint64_t second;  // an item's stream 1 may begin
    __shared__ uint32_t tmem_base;
    __shared__ float2 sh_ml[2][2][128];  // by stream, half and row: maximum and sum
    __shared__ float sh_mx[2][2][128];
    __shared__ int sh_bad[17];  // a node's V holds NaN or infinities: by item, and (16) any so far in the odd tiles' ring
    const ds_cuda_tree_attention_t &d = a.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    sa_warm<HD>(a);
    if (tid == TC_SOFTMAX) {
        for (int u = 0; u < NU; u++) {
            mbar_init(&full[u], 32);
            mbar_init(&empty[u], S::DUAL ? 2 : 1);
        }
        mbar_init(&qfull, TC_SOFTMAX / 32);
        mbar_init(&second, 8);
        for (int w = 0; w < 2; w++) {
            mbar_init(&sfull[w][0], 1);
            mbar_init(&sfull[w][1], 1);
            mbar_init(&pfull[w][0], 8);
            mbar_init(&pfull[w][1], 8);
            mbar_init(&pvdone[w], 1);
            mbar_init(&odone[w], 1);
            mbar_init(&drain[w], 1);
        }
        mbar_fence_init();
    }
    if (tid < 17) sh_bad[tid] = 0;
    if (warp == (TC_SOFTMAX + TC_PRODUCERS) / 32) tmem_alloc(&tmem_base, 512);
    SaCursor cu;
    int tiles;
    if (!sa_begin<KT, false, TC_THREADS>(a, cu, tiles)) tiles = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(DS_FULL, tmem_base, 0);
    bool ok = tiles > 0;
    // tiles of the run's next item that are this CTA's
    auto here = [&](int left) { return min(left, cu.s.tiles - cu.t); };
    auto to_next_item = [&]() {
        cu.t = cu.s.tiles - 1;
        sa_next<KT>(a, cu);
    };

    constexpr int MMA_WARP = (TC_SOFTMAX + TC_PRODUCERS) / 32;
    if (warp >= TC_SOFTMAX / 32 && warp < MMA_WARP) {
        // ---- producers: a warp a ring; whole tiles by TMA, others 16 bytes a
        // lane at a time ----
        const int rg = __shfl_sync(DS_FULL, warp - TC_SOFTMAX / 32, 0), cc = lane % CH, rr = lane / CH;
        constexpr int RS = 32 / CH;
        int item = 0, units = 0;  // units so far
        // (rows that one row tile reads once do not push the parts out of L2)
        uint64_t policy;
        if (a.row_tiles == 1) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
        auto load = [&](int t, int kv) {
            const int slot = rg * S::RING + units % S::RING;
            ok = __all_sync(DS_FULL, ok && tc_wait(&empty[slot], (units / S::RING & 1) ^ 1, a.err));
            if (!ok) return;
            units++;
            uint8_t *const unit = ring + slot * S::UNIT;
            if (args.mapped && (cu.t + t + 1) * KT <= cu.s.len) {
                if (elect_one()) {
                    const int *const dim = args.dim[kv];
                    const int r0 = (cu.t + t) * KT;
                    const int y = dim[0] == 1 ? r0 : dim[1] == 1 ? cu.g : cu.b, z = dim[0] == 2 ? r0 : dim[1] == 2 ? cu.g : cu.b,
                              v = dim[0] == 3 ? r0 : dim[1] == 3 ? cu.g : cu.b;
                    mbar_arrive_n(&full[slot], 31);
                    mbar_expect_tx(&full[slot], S::UNIT);
#pragma unroll
                    for (int k = 0; k < HD / 64; k++)
                        tma_load_4d(unit + k * S::SUB, &args.map[kv], 64 * k, y, z, v, &full[slot], policy);
                }
                __syncwarp();
                return;
            }
            SaCursor c = cu;
            c.t += t;
            const SaTile src = sa_tile<KT>(d, c);
            const uint16_t *x = src.base[kv][0] + rr * src.step[kv] + 8 * cc;
            const uint32_t dst = smem_u32(unit) + (cc >> 3) * S::SUB;
            auto at = [&](int r) { return (uint32_t)(r * 128 + (((cc & 7) ^ (r & 7)) << 4)); };
            if (src.valid >= KT) {
#pragma unroll 8
                for (int r = rr; r < KT; r += RS, x += RS * src.step[kv]) cp16(dst + at(r), x);
            } else {
#pragma unroll 8
                for (int r = rr; r < KT; r += RS, x += RS * src.step[kv]) cp16(dst + at(r), r < src.valid ? x : d.q, r < src.valid);
            }
            if (src.node && kv) {
                // A node's V may hold NaN or infinities that some rows must not
                // see, and 0 * NaN would spread through the product: they are
                // zeroed here, and added to the results of the rows that attend
                // them when those are written. (Every item has units in ring 0,
                // which is thus fewer than 16 items ahead. Ring 1 of the odd
                // tiles runs past any number of one-tile items: its flag stays
                // set, and the later items' nodes are looked through.)
                cp_commit();
                cp_wait<0>();
                // (an exponent of all ones carries into the bit above it)
                constexpr uint32_t E = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
                auto scan = [&](auto found) {
#pragma unroll 4
                    for (int r = rr; r < min(KT, src.valid); r += RS) {
                        uint4 *const v = reinterpret_cast<uint4 *>(unit + (cc >> 3) * S::SUB + at(r));
                        const uint4 u = *v;
                        if ((((u.x & E) + ONE) | ((u.y & E) + ONE) | ((u.z & E) + ONE) | ((u.w & E) + ONE)) & 0x80008000u) found(v, u);
                    }
                };
                bool bad = false;
                scan([&](uint4 *, uint4) { bad = true; });
                if (bad) {
                    scan([&](uint4 *v, uint4 u) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            uint32_t &x = (&u.x)[k];
                            const uint32_t top = ((x & E) + ONE) & 0x80008000u;
                            x &= ~((top >> 15) * 0xffffu);
                        }
                        *v = u;
                    });
                    *reinterpret_cast<volatile int *>(&sh_bad[S::DUAL || rg == 0 ? item & 15 : 16]) = 1;
                }
                fence_proxy_async();
                mbar_arrive(&full[slot]);
            } else {
                cp_arrive(&full[slot]);
            }
        };
        for (int left = tiles; left > 0 && ok; item++) {
            const int n = here(left);
            if (S::DUAL) {
                for (int t = 0; t < n; t++) load(t, rg);
            } else {
                const int mine = (n - rg + 1) >> 1;
                for (int place = 0; place < 2 * mine; place++) {
                    int kv;
                    const int t = S::at(place, mine, kv);
                    load(2 * t + rg, kv);
                }
            }
            left -= n;
            if (left > 0) to_next_item();
        }
        cp_commit();
        cp_wait<0>();
        if (!ok)  // a wait gave up: what was issued arrives before the memory goes
            for (int u = max(0, units - S::RING); u < units; u++) tc_wait(&full[rg * S::RING + u % S::RING], u / S::RING & 1, nullptr);
    } else if (warp >= MMA_WARP) {
        // ---- stream w's products: the warp waits, one lane issues ----
        const int w = __shfl_sync(DS_FULL, warp - MMA_WARP, 0);
        constexpr uint32_t is = F16 ? idesc_f16_f32(128, KT) : idesc_bf16_f32(128, KT);
        constexpr uint32_t ip = (F16 ? idesc_f16_f32(128, HD) : idesc_bf16_f32(128, HD)) | (1u << 16);  // V is MN-major
        const uint32_t ring_k = (((smem_u32(ring) >> 4) & 0x3fffu) | (1u << 16));
        const uint32_t ring_v = (((smem_u32(ring) >> 4) & 0x3fffu) | ((S::SUB >> 4) << 16));
        const uint32_t q = ((smem_u32(smem + (S::DUAL ? w * S::QBLOCK : 0)) >> 4) & 0x3fffu) | (1u << 16);
        const uint32_t ts = tmem + S::TS + w * 2 * KT, to = tmem + S::TO + w * HD;
        int done = 0;  // this stream's tiles before the item
        auto wait = [&](uint64_t *bar, uint32_t ph) { ok = __all_sync(DS_FULL, ok && tc_wait(bar, ph, a.err)); };
        // unit u of ring rg, of the item's tile t
        auto take = [&](int rg, int u, int t) {
            const int s = rg * S::RING + u % S::RING;
            wait(&full[s], u / S::RING & 1);
            // copies that are not TMA's are ordinary writes, the products'
            // reads are not
            if (!args.mapped || (cu.t + t + 1) * KT > cu.s.len) fence_proxy_async();
            return s;
        };
        for (int left = tiles, item = 0; left > 0 && ok; item++) {
            const int n = here(left), steps = S::DUAL ? n : (n - w + 1) >> 1;
            auto qk = [&](int j) {
                const int t = S::DUAL ? j : 2 * j + w, buf = (done + j) & 1;
                const int s = S::DUAL ? take(0, done + j, t) : take(w, 2 * done + S::place_k(j), t);
                if (!ok) return;
                tc_fence_after();
                const uint32_t k = ring_k + s * (S::UNIT >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int x = 0; x < HD / 16; x++)
                        umma_ss(ts + buf * KT, q + (x / 4) * (S::QSUB >> 4) + 2 * (x % 4), k + (x / 4) * (S::SUB >> 4) + 2 * (x % 4),
                                TC_DHI, is, x > 0);
                    umma_commit(&sfull[w][buf]);
                    umma_commit(&empty[s]);
                }
                __syncwarp();
            };
            wait(&qfull, item & 1);
            for (int j = 0; j < min(2, steps) && ok; j++) qk(j);
            for (int j = 0; j < steps && ok; j++) {
                const int t = S::DUAL ? j : 2 * j + w, buf = (done + j) & 1;
                const int s = S::DUAL ? take(1, done + j, t) : take(w, 2 * done + S::place_v(j, steps), t);
                wait(&pfull[w][buf], (done + j) >> 1 & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t v = ring_v + s * (S::UNIT >> 4);
                if (elect_one()) {
                    if (j == 0) umma_ts<0>(to, ts + buf * KT, v, TC_DHI, ip);
                    else umma_ts<1>(to, ts + buf * KT, v, TC_DHI, ip);
#pragma unroll
                    for (int x = 1; x < KT / 16; x++) umma_ts<1>(to, ts + buf * KT + 8 * x, v + 128 * x, TC_DHI, ip);
                    umma_commit(&pvdone[w]);
                    umma_commit(&empty[s]);
                    if (j + 1 == steps) umma_commit(&odone[w]);
                }
                __syncwarp();
                if (j + 2 < steps) {  // S over this P, once the product has read it
                    wait(&pvdone[w], (done + j) & 1);
                    if (ok) qk(j + 2);
                }
            }
            // (a stream without a tile says so: the item's end waits for both)
            if (steps == 0 && lane == 0) mbar_arrive(&odone[w]);
            done += steps;
            left -= n;
            if (left > 0) to_next_item();
        }
        if (!ok && tiles > 0) {  // a wait gave up: what was issued ends before the memory goes
            if (elect_one()) umma_commit(&drain[w]);
            __syncwarp();
            tc_wait(&drain[w], 0, nullptr);
        }
    } else {
        // ---- softmax: row i of stream w, keys (and dimensions) of half h ----
        const int w = warp >> 3, h = warp >> 2 & 1, i = 32 * (warp & 3) + lane, pair = 1 + 4 * w + (warp & 3);
        const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t to = tl + S::TO + w * HD;
        const float c = fabsf(a.scale2);
        const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;  // the sign goes to the queries
        constexpr int PARTS = S::DUAL ? 2 : 4;                    // threads of a row
        const int part = S::DUAL ? h : 2 * w + h;
        int item = 0, done = 0;  // this stream's tiles before the item
        // the queries of an item's rows, swizzled as K is (all loads first:
        // stores in between would hold them up)
        constexpr int QN = CH / PARTS;
        uint4 qu[QN];
        auto q_load = [&]() {
            const int row = cu.rt * S::RT + (S::DUAL ? w * 128 : 0) + i;
            const uint4 *const q = reinterpret_cast<const uint4 *>((const uint16_t *)d.q + cu.b * d.q_stride[0] + (row / a.group) * d.q_stride[1] +
                                                                   (cu.g * a.group + row % a.group) * d.q_stride[2]) + part * QN;
#pragma unroll
            for (int k = 0; k < QN; k++) qu[k] = row < a.rows ? q[k] : make_uint4(0, 0, 0, 0);
        };
        auto q_store = [&]() {
            uint8_t *const q = smem + (S::DUAL ? w * S::QBLOCK : 0) + i * 128;
#pragma unroll
            for (int k = 0; k < QN; k++) {
                const int ch = part * QN + k;
                qu[k].x ^= flip, qu[k].y ^= flip, qu[k].z ^= flip, qu[k].w ^= flip;
                *reinterpret_cast<uint4 *>(q + (ch >> 3) * S::QSUB + (((ch & 7) ^ (i & 7)) << 4)) = qu[k];
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&qfull);
        };
        for (int left = tiles; left > 0 && ok; item++) {
            const int n = here(left);
            const bool whole = cu.t == 0, end = cu.t + n == cu.s.tiles;
            const int row = cu.rt * S::RT + (S::DUAL ? w * 128 : 0) + i, nd = row / a.group, head = cu.g * a.group + row % a.group;
            const bool used = row < a.rows && nd < cu.s.cnt;
            if (item == 0) {
                q_load();
                q_store();
            }
            const uint64_t *const words = d.mask + ((size_t)cu.b * d.n_nodes + (used ? nd : 0)) * a.words;
            // the mask's word for this stream's next tile of nodes
            auto word_of = [&](int k) { return used && k * KT < cu.s.cnt ? (uint32_t)(words[k] >> (32 * h)) : 0u; };
            int nodes0 = max(0, cu.s.cache_tiles - cu.t);
            if (!S::DUAL) nodes0 += (nodes0 ^ w) & 1;
            uint32_t word = word_of(cu.t + nodes0 - cu.s.cache_tiles);
            float m = -__FLT_MAX__, l = 0.f;
            int step = done;
            // (after a wait that gave up: on without waiting, through every
            // barrier, to the item's end)
            auto tile = [&](auto masks, int t) {
                constexpr bool MASKED = decltype(masks)::value;
                const int buf = step & 1;
                const uint32_t ts = tl + S::TS + (2 * w + buf) * KT;
                uint32_t see = ~0u;
                if (MASKED) {
                    const bool node = cu.t + t >= cu.s.cache_tiles;
                    const int r0 = (node ? cu.t + t - cu.s.cache_tiles : cu.t + t) * KT;
                    const int valid = (node ? cu.s.cnt : cu.s.len) - r0 - 32 * h;  // of this half's keys
                    see = valid >= 32 ? ~0u : valid > 0 ? (1u << valid) - 1 : 0;
                    if (node) {
                        see &= word;
                        word = word_of(r0 / KT + STEP);
                    }
                }
                ok = ok && tc_wait(&sfull[w][buf], step >> 1 & 1, a.err);
                __syncwarp();
                tc_fence_after();
                float v[32], lt;
                uint32_t pk[16];
                tmem_ld32(ts + 32 * h, v);
                // the row's maximum over both halves (and what m was)
                auto look = [&]() {
                    float mt = m;
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!MASKED || (see >> e & 1)) mt = fmaxf(mt, v[e]);
                    sh_mx[w][h][i] = mt;
                    bar_sync(pair, 64);
                    m = fmaxf(mt, sh_mx[w][h ^ 1][i]);
                };
                // weights of the row's keys with m, their sum, and packed in pairs
                auto weigh = [&]() {
                    const float mc = fmaxf(m * c, -__FLT_MAX__) - sa_lift<F16>();
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        v[e] = ex2(__fmaf_rn(v[e], c, -mc));
                        if (MASKED) v[e] = see >> e & 1 ? v[e] : 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        s[e & 3] += v[2 * e] + v[2 * e + 1];
                        pk[e] = pack2<F16>(v[2 * e], v[2 * e + 1]);
                    }
                    lt = (s[0] + s[1]) + (s[2] + s[3]);
                };
                if (t < STEP) {
                    // An item's stream 1 begins when stream 0 has its first
                    // weights: half a step apart, one's waits, loads and stores
                    // run beside the other's exponentials.
                    look();
                    if (w) ok = ok && tc_wait(&second, item & 1, a.err);
                    __syncwarp();
                    weigh();
                    if (!w && lane == 0) mbar_arrive(&second);
                } else {
                    // The sum tells whether m still serves: a tile that passes
                    // 2^10 in either half of any of the 32 rows is done again
                    // with the true maxima. (So a weight is at most 2^10, and m
                    // never above the row's maximum. FP16: 2^15, which is 2^8
                    // times 2^SA_LIFT.)
                    weigh();
                    if (bar_or(pair, 64, !(lt <= (F16 ? 32768.f : 1024.f)))) {
                        const float was = m;
                        tmem_ld32(ts + 32 * h, v);
                        look();
                        const float f = m > was ? ex2((was - m) * c) : 1.f;
                        weigh();
                        l *= f;
                        // (the last tile's product has to be in O)
                        ok = ok && tc_wait(&pvdone[w], (step - 1) & 1, a.err);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int k = 0; k < HD / 2; k += 16) {
                            float y[16];
                            tmem_ld16(to + h * (HD / 2) + k, y);
#pragma unroll
                            for (int e = 0; e < 16; e++) y[e] *= f;
                            tmem_st16f(to + h * (HD / 2) + k, y);
                        }
                    }
                }
                l += lt;
                tmem_st16(ts + 16 * h, pk);  // over S, which both halves have read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[w][buf]);
                step++;
            };
            const int plain = min(n, cu.s.len / KT - cu.t);  // tiles without a mask
            int t = S::DUAL ? 0 : w;
            for (; t < plain; t += STEP) tile(std::false_type(), t);
            for (; t < n; t += STEP) tile(std::true_type(), t);
            // the results: a stream's own rows, or the streams' joined; a row's
            // threads take a share of the dimensions each
            const bool both = S::DUAL || n > 1;
            done = step;
            // the next item's queries come in while this one's products end,
            // and go to shared memory as soon as they have: its first S are
            // ready when this one's results are written. (Its first O waits
            // for weights, which come after the barrier below.)
            const SaCursor it = cu;
            left -= n;
            if (left > 0) {
                to_next_item();
                q_load();
            }
            sh_ml[w][h][i] = make_float2(fmaxf(m * c, -__FLT_MAX__) - sa_lift<F16>(), l);
            if (ok) ok = tc_wait(&odone[0], item & 1, a.err);
            if (ok) ok = tc_wait(&odone[1], item & 1, a.err);
            ok = __all_sync(DS_FULL, ok);
            if (ok && left > 0) q_store();
            tc_fence_after();
            bar_sync(TC_ALL, TC_SOFTMAX);
            float mm, ll, f0 = 1.f, f1 = 0.f;
            if (S::DUAL) {
                mm = sh_ml[w][0][i].x;
                ll = sh_ml[w][0][i].y + sh_ml[w][1][i].y;
            } else {
                const float2 x = sh_ml[0][0][i], y = both ? sh_ml[1][0][i] : make_float2(-__FLT_MAX__, 0.f);
                mm = fmaxf(x.x, y.x);
                f0 = ex2(x.x - mm);
                f1 = ex2(y.x - mm);
                ll = (x.y + sh_ml[0][1][i].y) * f0;
                if (both) ll += (y.y + sh_ml[1][1][i].y) * f1;
            }
            if (ok) {
                const bool alone = whole && end, none = !used || ll == 0.f;
                const float inv = alone ? (none ? 0.f : 1.f / ll) : 1.f;
                const bool bad = (*reinterpret_cast<volatile int *>(&sh_bad[item & 15]) | (S::DUAL ? 0 : *reinterpret_cast<volatile int *>(&sh_bad[16]))) != 0;
                const size_t slot = (size_t)blockIdx.x * 2 + whole;
                const int r = (S::DUAL ? w * 128 : 0) + i;
#pragma unroll 1
                for (int k = 0; k < HD / PARTS; k += 16) {
                    const int c0 = part * (HD / PARTS) + k;
                    __syncwarp();
                    float v[16];
                    if (S::DUAL) {
                        tmem_ld16(to + c0, v);
                    } else {
                        tmem_ld16(tl + S::TO + c0, v);
                        if (both) {
                            float y[16];
                            tmem_ld16(tl + S::TO + HD + c0, y);
#pragma unroll
                            for (int e = 0; e < 16; e++) v[e] = v[e] * f0 + y[e] * f1;
                        }
                    }
                    if (bad && used)  // see the producers
                        for (int j = 0; j < it.s.cnt; j++)
                            if (words[j >> 6] >> (j & 63) & 1) {
                                const uint16_t *x = (const uint16_t *)d.tree_v + it.b * d.tree_v_stride[0] +
                                                    it.g * d.tree_v_stride[1] + j * d.tree_v_stride[2] + c0;
#pragma unroll
                                for (int e = 0; e < 16; e++) {
                                    const float y = F16 ? __half2float(__ushort_as_half(x[e])) : __uint_as_float((uint32_t)x[e] << 16);
                                    if (!isfinite(y)) v[e] += y;
                                }
                            }
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = alone && none ? 0.f : v[e] * inv;
                    if (row < a.rows) {
                        if (alone) {
                            uint16_t *o = (uint16_t *)d.out + it.b * d.out_stride[0] + nd * d.out_stride[1] + head * d.out_stride[2] + c0;
#pragma unroll
                            for (int e = 0; e < 16; e += 8)
                                *reinterpret_cast<uint4 *>(o + e) = make_uint4(pack2<F16>(v[e], v[e + 1]), pack2<F16>(v[e + 2], v[e + 3]),
                                                                               pack2<F16>(v[e + 4], v[e + 5]), pack2<F16>(v[e + 6], v[e + 7]));
                        } else {
                            float *const o = a.part + (slot * HD + c0) * S::RT + r;  // [dimension][row]
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e * S::RT] = v[e];
                        }
                    }
                }
                if (row < a.rows && (S::DUAL ? h == 0 : part == 0)) {
                    if (!alone) a.ml[slot * S::RT + r] = make_float2(mm, ll);
                    else if (d.lse)
                        d.lse[((size_t)it.b * d.n_nodes + nd) * d.n_heads + head] = none ? -INFINITY : (mm + log2f(ll)) * 0.69314718f;
                }
            }
            // every reader of sh_ml, sh_bad and O is done; all go on or none
            tc_fence_before();
            ok = bar_and(TC_ALL, TC_SOFTMAX, ok);
            if (tid == 0) sh_bad[item & 15] = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// The items that several CTAs had parts of. Parts are [row][dimension] with
// HD / 4 threads a row, one row each, or (WIDE) all on one row, where rows are
// few and parts may be many. The parts of sa_many_kernel are [dimension][row]:
// a CTA takes 32 rows, a warp an eighth of the dimensions; or (WIDE) 32 rows
// and 16 dimensions, a warp every eighth part.
constexpr int SJ_THREADS = 256, SJ_WARPS = SJ_THREADS / 32;
template <class S> struct SaMade {
    static constexpr bool by_dimension = false;
};
template <int HD, bool DUAL, int QT> struct SaMade<SaMany<HD, DUAL, QT>> {
    static constexpr bool by_dimension = true;
};
// Rows a CTA takes, and CTAs of an item.
template <class S> constexpr int sj_rows(bool wide) {
    return SaMade<S>::by_dimension ? 32 : wide ? 1 : std::min(S::RT, SJ_THREADS / (S::HD / 4));
}
template <class S> constexpr int sj_ctas(bool wide) {
    return S::RT / sj_rows<S>(wide) * (SaMade<S>::by_dimension && wide ? S::HD / 16 : 1);
}

// Loads that stay where they are written: the compiler would move each to its
// use, which makes the parts' latencies follow one another.
__device__ __forceinline__ float sj_ld(const float *p) {
    float v;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float2 sj_ld2(const float2 *p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 sj_ld4(const float *p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
template <class S, bool WIDE>
__global__ void __launch_bounds__(SJ_THREADS) sa_join_kernel(const __grid_constant__ SaArgs a) {
    constexpr int HD = S::HD, KT = S::KT, RT = S::RT;
    constexpr bool BYD = SaMade<S>::by_dimension;
    __shared__ int sh_scan[SJ_WARPS], sh_off;
    const ds_cuda_tree_attention_t &d = a.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y;
    const int chunk = (d.batch + SJ_THREADS - 1) / SJ_THREADS;
    const int b0 = min(d.batch, tid * chunk), b1 = min(d.batch, b0 + chunk);
    int at;
    const SaSeq s = sa_seq<KT>(d, b);
    const int total = sa_scan<KT, SJ_THREADS>(a, b0, b1, sa_seq<KT>(d, min(b0, d.batch - 1)), sh_scan, &at);
    if (b0 <= b && b < b1) {
        for (int y = b0; y < b; y++) at += sa_seq<KT>(d, y).tiles * a.per_seq;
        sh_off = at;
    }
    __syncthreads();
    const SaCut cut(total, a.ctas);
    // this thread's row and first dimension, and the parts it takes
    const int item = blockIdx.x / sj_ctas<S>(WIDE), in = blockIdx.x % sj_ctas<S>(WIDE);
    const int grp = BYD ? warp : tid / (HD / 4), groups = WIDE ? (BYD ? SJ_WARPS : SJ_THREADS / (HD / 4)) : 1;
    constexpr int VN = BYD ? (WIDE ? 16 : HD / SJ_WARPS) : 4;
    const int r = BYD ? (WIDE ? in / (HD / 16) : in) * 32 + lane : WIDE ? in : in * sj_rows<S>(false) + grp;  // (>= RT: none)
    const int c = BYD ? (WIDE ? in % (HD / 16) * 16 : warp * VN) : 4 * (tid % (HD / 4));
    const int x0 = sh_off + item * s.tiles, c0 = cut.cta_of(x0), c1 = cut.cta_of(x0 + s.tiles - 1);
    const int row = r < RT ? item % a.row_tiles * RT + r : a.rows, g = item / a.row_tiles;
    pdl_wait();
    if (c0 == c1) return;
    float m = -__FLT_MAX__, l = 0.f, o[VN] = {};
    if (row < a.rows) {
        // four parts at a time, all their loads first
        constexpr int AHEAD = 4;
        for (int k0 = c0 + (WIDE ? grp : 0); k0 <= c1; k0 += AHEAD * groups) {
            float2 ml[AHEAD];
            float v[AHEAD][VN];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int cc = min(k0 + k * groups, c1);
                const size_t slot = (size_t)cc * 2 + (cc == c0);
                ml[k] = sj_ld2(a.ml + slot * RT + r);
                if (BYD) {
#pragma unroll
                    for (int e = 0; e < VN; e++) v[k][e] = sj_ld(a.part + (slot * HD + c + e) * RT + r);
                } else {
                    const float4 u = sj_ld4(a.part + (slot * RT + r) * HD + c);
                    v[k][0] = u.x, v[k][1] = u.y, v[k][2] = u.z, v[k][3] = u.w;
                }
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) mn = fmaxf(mn, ml[k].x);
            const float f = ex2(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int e = 0; e < VN; e++) o[e] *= f;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const bool is = k0 + k * groups <= c1;
                const float e2 = ex2(ml[k].x - mn);
                l += is ? ml[k].y * e2 : 0.f;
#pragma unroll
                for (int e = 0; e < VN; e++) o[e] += is ? v[k][e] * e2 : 0.f;
            }
        }
    }
    if (!WIDE) {
        if (row >= a.rows) return;
        if constexpr (BYD) {  // 16-bit types: a thread's dimensions in 16-byte stores
            const int nd = row / a.group, head = g * a.group + row % a.group;
            const bool none = nd >= s.cnt || l == 0.f;
            const float inv = 1.f / l;
            constexpr bool F16 = S::QT == DS_CUDA_SPEC_F16;
            uint4 *const out = reinterpret_cast<uint4 *>((uint16_t *)d.out + b * d.out_stride[0] + nd * d.out_stride[1] + head * d.out_stride[2] + c);
#pragma unroll
            for (int e = 0; e < VN; e++) o[e] = none ? 0.f : o[e] * inv;
#pragma unroll
            for (int e = 0; e < VN; e += 8)
                out[e / 8] = make_uint4(pack2<F16>(o[e], o[e + 1]), pack2<F16>(o[e + 2], o[e + 3]), pack2<F16>(o[e + 4], o[e + 5]),
                                        pack2<F16>(o[e + 6], o[e + 7]));
            if (d.lse && c == 0)
                d.lse[((size_t)b * d.n_nodes + nd) * d.n_heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.69314718f;
        } else {
            sa_finish(a, b, g, row, s.cnt, c, m, l, o);
        }
        return;
    }
    // the groups' results, in order
    const int n = min(groups, c1 - c0 + 1);
    if (BYD) {
        __shared__ float sh_o[BYD ? SJ_WARPS : 1][32][17];
        __shared__ float2 sh_ml[BYD ? SJ_WARPS : 1][32];
        if (warp < n) {
            sh_ml[BYD ? warp : 0][lane] = make_float2(m, l);
#pragma unroll
            for (int e = 0; e < VN; e++) sh_o[BYD ? warp : 0][lane][e % 16] = o[e];
        }
        __syncthreads();
        const int rr = tid >> 2, cc = 4 * (tid & 3), out = row - lane + rr;
        if (rr >= 32 || out >= a.rows) return;
        float mm = -__FLT_MAX__, ll = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < n; k++) mm = fmaxf(mm, sh_ml[k][rr].x);
        for (int k = 0; k < n; k++) {
            const float f = ex2(sh_ml[k][rr].x - mm);
            ll += sh_ml[k][rr].y * f;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += sh_o[k][rr][cc + e] * f;
        }
        sa_finish(a, b, g, out, s.cnt, c + cc, mm, ll, v);
    } else {
        __shared__ float4 sh_o[SJ_THREADS];
        __shared__ float2 sh_ml[SJ_THREADS];
        sh_o[tid] = make_float4(o[0], o[1], o[2], o[3]);
        sh_ml[tid] = make_float2(m, l);
        __syncthreads();
        if (grp || row >= a.rows) return;
        float mm = -__FLT_MAX__, ll = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < n; k++) mm = fmaxf(mm, sh_ml[k * (HD / 4) + tid].x);
        for (int k = 0; k < n; k++) {
            const float2 ml = sh_ml[k * (HD / 4) + tid];
            sa_add(v, ll, sh_o[k * (HD / 4) + tid], ml.y, ex2(ml.x - mm));
        }
        sa_finish(a, b, g, row, s.cnt, c, mm, ll, v);
    }
}


// Calls whose items are few enough for a cluster each in one wave, with at
// most 8 tiles a CTA, are joined in the clusters: one launch, no workspace.
// Their tiles are bounded by the cache's room, the lengths not being known
// here. Others take the list. How many clusters are a wave the runtime says: a
// cluster is of one GPC, whose SMs need not be a multiple of its CTAs (one node,
// 16 heads, 662 tokens, F32: two waves of 16 CTAs take 12.7 us, one of 8 CTAs
// 8.7 us). Clusters have 16 CTAs, or 8 with eight rows a tile (with 16, F32, 32 rows of 10 heads over 662 tokens take 13.7 us in
// clusters of 8 and 12.5 in the list).
// (One stream, 10 heads, 662 tokens, F32 in two planes: one node takes 7.3 us
// on the GPU against 8.0, and the call 7 us of the host's time instead of 13.)
static long long sa_most_tiles(const ds_cuda_tree_attention_t *d, int kt) {
    return ((long long)d->kv_max + kt - 1) / kt + (d->n_nodes + kt - 1) / kt;
}
// A kernel's attributes, once per device (of the first 64).
template <class S, bool CLUSTER> static cudaError_t sa_attributes(int device) {
    static std::atomic<uint64_t> ready;
    if (device < 64 && ready.load() >> device & 1) return cudaSuccess;
    const void *f;
    if constexpr (SaMade<S>::by_dimension) f = (const void *)sa_many_kernel<S>;
    else f = (const void *)sa_few_kernel<S, CLUSTER>;
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e == cudaSuccess && CLUSTER) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < 64) ready.fetch_or(1ull << device);
    return e;
}
template <class S> static cudaLaunchConfig_t sa_cluster_config(cudaLaunchAttribute &attr, dim3 grid, int n, cudaStream_t st) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = n;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(SA_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cfg;
}
// Clusters of n CTAs that the (current) device holds at once; asked once per
// device of the first 64. 0 where it cannot say, which leaves the list.
template <class S> static int sa_wave(int device, int n) {
    static std::atomic<int> known[64][2];  // 1 + the answer, of 8 and of 16 CTAs
    std::atomic<int> *const k = device < 64 ? &known[device][n > 8] : nullptr;
    if (const int v = k ? k->load() : 0) return v - 1;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = sa_cluster_config<S>(attr, dim3(n), n, nullptr);
    int most = 0;
    if (sa_attributes<S, true>(device) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&most, (const void *)sa_few_kernel<S, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        most = 0;
    }
    if (k) k->store(1 + most);
    return most;
}
template <class S> static int sa_clusters(const ds_cuda_tree_attention_t *d, long long items, int device) {
    for (int n = SA_CLUSTER; n >= (S::RT == 8 ? 8 : SA_CLUSTER); n /= 2)
        if (sa_most_tiles(d, S::KT) <= 8 * n && items <= sa_wave<S>(device, n)) return n;
    return 0;
}

// The cache's K or V as a tensor map: the dimensions after the head's own in
// the order of their strides. False where the strides allow none.
static bool sa_map(const ds_cuda_tree_attention_t &d, int kv, int kt, CUtensorMap *map, int (&dim)[3]) {
    const int64_t *const s = kv ? d.v_stride : d.k_stride;
    const int64_t step[3] = {s[2], s[1], s[0]};
    const int extent[3] = {d.kv_max, d.n_kv_heads, d.batch};
    if (d.kv_max < kt) return false;
    int order[3] = {0, 1, 2};
    auto key = [&](int i) { return extent[i] > 1 ? step[i] : INT64_MAX; };  // a stride that is never used goes last
    std::sort(order, order + 3, [&](int x, int y) { return key(x) < key(y); });
    cuuint64_t dims[4] = {(cuuint64_t)d.head_dim}, strides[3];
    cuuint32_t box[4] = {64, 1, 1, 1}, one[4] = {1, 1, 1, 1};
    for (int k = 0; k < 3; k++) {
        const int i = order[k];
        const int64_t most = k ? (int64_t)(strides[k - 1] * dims[k]) : 2 * d.head_dim;
        if (extent[i] > 1 && (step[i] <= 0 || 2 * step[i] >= (int64_t)1 << 40)) return false;
        strides[k] = extent[i] > 1 ? 2 * step[i] : (most + 15) / 16 * 16;
        if (strides[k] >= (cuuint64_t)1 << 40) return false;
        dims[k + 1] = extent[i];
        dim[i] = k + 1;
        if (i == 0) box[k + 1] = kt;
    }
    const EncodeTiledFn enc = encode_tiled();
    return enc && enc(map, d.type == DS_CUDA_SPEC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                      const_cast<void *>(kv ? d.v : d.k), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class S> struct SaRun {
    static int clusters(const ds_cuda_tree_attention_t *d, long long items, int device) {
        if constexpr (SaMade<S>::by_dimension) return 0;
        else return sa_clusters<S>(d, items, device);
    }
    static size_t workspace(const SaArgs &a) {
        // two parts a CTA, then their maxima and sums
        return a.cluster ? 0 : (size_t)a.sms * S::PER_SM * 2 * S::RT * (S::HD * 4 + 8);
    }
    static cudaError_t run(SaArgs a, int device, cudaStream_t st) {
        void *args[] = {&a};
        if constexpr (!SaMade<S>::by_dimension) if (a.cluster) {
            const cudaError_t e = sa_attributes<S, true>(device);
            if (e != cudaSuccess) return e;
            cudaLaunchAttribute attr;
            const cudaLaunchConfig_t cfg = sa_cluster_config<S>(attr, dim3(a.row_tiles * a.cluster, a.d.n_kv_heads, a.d.batch), a.cluster, st);
            return cudaLaunchKernelExC(&cfg, (const void *)sa_few_kernel<S, true>, args);
        }
        a.ctas = a.sms * S::PER_SM;
        a.part = (float *)a.d.workspace;
        a.ml = (float2 *)(a.part + (size_t)a.ctas * 2 * S::RT * S::HD);
        cudaError_t e = sa_attributes<S, false>(device);
        if (e != cudaSuccess) return e;
        if constexpr (SaMade<S>::by_dimension) {
            SaManyArgs many = {};
            many.a = a;
            many.mapped = sa_map(a.d, 0, S::KT, &many.map[0], many.dim[0]) && sa_map(a.d, 1, S::KT, &many.map[1], many.dim[1]);
            sa_many_kernel<S><<<a.ctas, TC_THREADS, S::SMEM, st>>>(many);
        } else {
            sa_few_kernel<S, false><<<a.ctas, SA_THREADS, S::SMEM, st>>>(a);
        }
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        const bool wide = (long long)a.d.batch * a.per_seq * S::RT <= a.sms * 8;
        return launch_ex(wide ? (const void *)sa_join_kernel<S, true> : (const void *)sa_join_kernel<S, false>,
                         dim3(a.per_seq * sj_ctas<S>(wide), a.d.batch), dim3(SJ_THREADS), 0, st, true, args);
    }
};

// f(instantiation) for a call, by its rows a KV head. F32 takes mma.sync, 8 or
// 16 rows at a time (on tcgen05 the planes' products could have columns of their
// own, but its sums round towards zero, so that they would have to be folded
// into F32 every few tiles: not built).
// Eight at a time also where each tile of eight has a cluster: one stream of 10
// heads, 16 rows, room for 1024 rows of which 662 are used, F32 9.1 us against
// 12.4, BF16 8.2 against 10.4; 20 rows of 8 KV heads, 1900 / 3900 tokens, F32
// 13.2 / 20.3 against 17.2 / 22.3; one head, 200 rows, 662 / 4000 tokens, F32
// 10.4 / 23.1 against 12.8 / 23.2.
// 16-bit types take mma.sync up to 16 rows, and for more where the call is brief: at
// most 8 tiles a CTA, by the cache's room. Else tcgen05, one block of 128 rows
// or two. BF16, mma.sync against tcgen05: 64 streams of 10 heads, up to 1325
// tokens, 8 / 16 / 24 / 48 rows 51 / 66 / 118 / 184 us against 79 / 80 / 81 /
// 84 us (but 8 streams on 8 KV heads, up to 8191 tokens, 16 rows 45 against
// 41); brief: one stream, 662 tokens, 32 / 64 / 128 rows 12 / 13 / 20 us
// against 20 / 20 / 27 us.
template <int HD, int QT, class F> static auto sa_pick16(int rows, bool apart, bool brief, F f) {
    return apart                 ? f(SaRun<SaFew<HD, 1, 1, QT>>())
           : rows <= 16 || brief ? f(SaRun<SaFew<HD, 2, 1, QT>>())
           : rows <= 128         ? f(SaRun<SaMany<HD, false, QT>>()) : f(SaRun<SaMany<HD, true, QT>>());
}
template <int HD, class F> static auto sa_pick_hd(const ds_cuda_tree_attention_t *d, const ds_cuda_ctx *c, F f) {
    constexpr int P = DS_CUDA_SPEC_F32;
    const int rows = d->n_nodes * (d->n_heads / d->n_kv_heads);
    using Few = SaFew<HD, 2, 1, DS_CUDA_SPEC_BF16>;
    const bool brief = (double)d->batch * d->n_kv_heads * ((rows + 15) / 16) * sa_most_tiles(d, SA_KT) <= 8.0 * c->sm_count * Few::PER_SM;
    using Eight = SaFew<HD, 1, 2, P>;
    const long long eights = (long long)d->batch * d->n_kv_heads * ((rows + 7) / 8);
    const bool apart = rows <= 8 || sa_clusters<Eight>(d, eights, c->device) > 0;
    if (d->type == DS_CUDA_SPEC_F16) return sa_pick16<HD, DS_CUDA_SPEC_F16>(rows, apart, brief, f);
    if (d->type == DS_CUDA_SPEC_BF16) return sa_pick16<HD, DS_CUDA_SPEC_BF16>(rows, apart, brief, f);
    if (d->k_lo || d->v_lo || d->tree_k_lo || d->tree_v_lo)
        return apart ? f(SaRun<SaFew<HD, 1, 2, P>>()) : f(SaRun<SaFew<HD, 2, 2, P>>());
    return apart ? f(SaRun<SaFew<HD, 1, 1, P>>()) : f(SaRun<SaFew<HD, 2, 1, P>>());
}
template <class F> static auto sa_pick(const ds_cuda_tree_attention_t *d, const ds_cuda_ctx *c, F f) {
    return d->head_dim == 64 ? sa_pick_hd<64>(d, c, f) : sa_pick_hd<128>(d, c, f);
}
template <class S> static S sa_shape(SaRun<S>) { return S(); }

// One CTA per sequence, one thread per node: a node's word bits are set by
// walking up its parents (kept in shared memory; at most n_nodes steps).
// Bound by the walk's latency: one tree of 16 takes 2.4 us, 64 random ones of
// 64 or 256 nodes 5.2 and 16 us, once a step for all layers.
__global__ void tree_mask_kernel(const int *parents, const int *nodes, int n, int words, uint64_t *mask, int *depth) {
    __shared__ int par[SA_MAX_NODES];
    const int b = blockIdx.x, i = threadIdx.x;
    const int cnt = nodes ? min(max(nodes[b], 0), n) : n;
    if (i < n) {
        const int p = parents[(size_t)b * n + i];
        par[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    if (i >= n) return;
    uint64_t w[SA_MAX_NODES / 64] = {};
    int deep = -1;
    for (int at = i < cnt ? i : -1; at >= 0; at = par[at]) {
#pragma unroll
        for (int k = 0; k < SA_MAX_NODES / 64; k++)
            if (at >> 6 == k) w[k] |= 1ull << (at & 63);
        deep++;
    }
#pragma unroll
    for (int k = 0; k < SA_MAX_NODES / 64; k++)
        if (k < words) mask[((size_t)b * n + i) * words + k] = w[k];
    if (depth) depth[(size_t)b * n + i] = max(deep, 0);
}

}  // namespace ds

using namespace ds;

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int sa_check(ds_cuda_ctx *c, const ds_cuda_tree_attention_t *d) {
    if (!d) return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: null descriptor");
    if (d->type < 0 || d->type > DS_CUDA_SPEC_F32) return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: type %d", d->type);
    if (d->batch < 0 || d->n_nodes <= 0 || d->n_nodes > SA_MAX_NODES || d->n_kv_heads <= 0 || d->n_heads <= 0 ||
        d->n_heads % d->n_kv_heads || (d->head_dim != 64 && d->head_dim != 128) || d->kv_max < 0 || d->kv_max > SA_MAX_KV)
        return ctx_fail(c, DS_CUDA_EINVAL,
                        "tree_attention: unsupported shape batch=%d n_nodes=%d n_heads=%d n_kv_heads=%d head_dim=%d "
                        "kv_max=%d (n_nodes <= %d, head_dim 64 or 128, n_heads a multiple of n_kv_heads, kv_max <= %d)",
                        d->batch, d->n_nodes, d->n_heads, d->n_kv_heads, d->head_dim, d->kv_max, SA_MAX_NODES, SA_MAX_KV);
    if (d->batch > 65535 || d->n_heads > 65535)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: batch and n_heads are at most 65535");
    return DS_CUDA_OK;
}

// The kernels' arguments but for what run() adds; `err` is told of a refusal.
static int sa_args(const ds_cuda_ctx *c, ds_cuda_ctx *err, const ds_cuda_tree_attention_t *d, SaArgs &a) {
    const int rc = sa_check(err, d);
    if (rc < 0) return rc;
    a.d = *d;
    a.words = (d->n_nodes + 63) / 64;
    a.group = d->n_heads / d->n_kv_heads;
    a.rows = d->n_nodes * a.group;
    const int rt = sa_pick(d, c, [](auto r) { return decltype(sa_shape(r))::RT; });
    a.row_tiles = (a.rows + rt - 1) / rt;
    a.per_seq = d->n_kv_heads * a.row_tiles;
    // (the list's places are 32-bit; its lengths are known on the device alone)
    const long long tiles = (long long)d->batch * a.per_seq * std::max(1ll, sa_most_tiles(d, SA_KT));
    if (tiles > INT32_MAX)
        return ctx_fail(err, DS_CUDA_EINVAL, "tree_attention: up to %lld tiles of %d keys and %d rows (< 2^31)", tiles, SA_KT, rt);
    a.sms = c->sm_count;
    a.cluster = sa_pick(d, c, [&](auto r) { return decltype(r)::clusters(d, (long long)d->batch * a.per_seq, c->device); });
    a.err = c->d_spec_err;
    a.scale2 = d->scale * 1.44269504f;
    return DS_CUDA_OK;
}

extern "C" size_t ds_cuda_tree_attention_workspace(const ds_cuda_ctx_t *c, const ds_cuda_tree_attention_t *d) {
    if (!c || !c->ok) return 0;
    const CtxDevice on(c);
    SaArgs a = {};
    if (sa_args(c, nullptr, d, a) < 0) return 0;
    return sa_pick(d, c, [&](auto r) { return decltype(r)::workspace(a); });
}

extern "C" int ds_cuda_tree_attention_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_attention_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    const CtxDevice on(c);
    SaArgs a = {};
    const int rc = sa_args(c, c, d, a);
    if (rc < 0 || d->batch == 0) return rc;
    if (!d->q || !d->out || !d->lens || !d->mask || !d->tree_k || !d->tree_v || (d->kv_max > 0 && (!d->k || !d->v)))
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: null pointer");
    const int qe = d->type == DS_CUDA_SPEC_F32 ? 4 : 2;
    const int g = d->n_kv_heads;
    const struct { const char *name; const void *p, *lo; const int64_t *s; int es, n1, n2; } ts[] = {
        {"q", d->q, nullptr, d->q_stride, qe, d->n_nodes, d->n_heads},
        {"out", d->out, nullptr, d->out_stride, qe, d->n_nodes, d->n_heads},
        {"k", d->k, d->k_lo, d->k_stride, 2, g, d->kv_max},
        {"v", d->v, d->v_lo, d->v_stride, 2, g, d->kv_max},
        {"tree_k", d->tree_k, d->tree_k_lo, d->tree_k_stride, 2, g, d->n_nodes},
        {"tree_v", d->tree_v, d->tree_v_lo, d->tree_v_stride, 2, g, d->n_nodes}};
    for (const auto &t : ts) {
        // the stride of a dimension of one element is never used
        const bool ok = (d->batch <= 1 || t.s[0] * t.es % 16 == 0) && (t.n1 <= 1 || t.s[1] * t.es % 16 == 0) &&
                        (t.n2 <= 1 || t.s[2] * t.es % 16 == 0);
        if (!ok || !aligned16(t.p) || !aligned16(t.lo))
            return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: %s: base and strides must be multiples of 16 bytes", t.name);
        if (t.lo && d->type != DS_CUDA_SPEC_F32)
            return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: %s has a lo plane, which only the F32 type takes", t.name);
    }
    const size_t need = sa_pick(d, c, [&](auto r) { return decltype(r)::workspace(a); });
    if (need && (!d->workspace || d->workspace_bytes < need || (reinterpret_cast<uintptr_t>(d->workspace) & 255)))
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: workspace of %zu bytes, 256-byte aligned, wanted", need);
    cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    const cudaError_t e = sa_pick(d, c, [&](auto r) { return decltype(r)::run(a, c->device, st); });
    if (e != cudaSuccess) cudaGetLastError();  // reported here, not by whoever asks next
    return ctx_cuda(c, e, "tree_attention launch");
}

extern "C" int ds_cuda_tree_attention_check(ds_cuda_ctx_t *c, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    const CtxDevice on(c);
    cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    unsigned err = 0;
    cudaError_t e = cudaMemcpyAsync(&err, c->d_spec_err, sizeof err, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return ctx_cuda(c, e, "tree_attention_check");
    // the count is never reset, or another stream's check would not see it
    const auto seen = c->spec_err_seen.find(st);
    if (err == (seen == c->spec_err_seen.end() ? 0 : seen->second)) return DS_CUDA_OK;
    c->spec_err_seen[st] = err;
    return ctx_fail(c, DS_CUDA_ETIMEOUT, "tree_attention: a bounded wait gave up");
}

extern "C" int ds_cuda_tree_mask_dev(ds_cuda_ctx_t *c, const int *parents, const int *nodes, int batch, int n_nodes,
                                     uint64_t *mask, int *depth, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (batch < 0 || n_nodes <= 0 || n_nodes > SA_MAX_NODES)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_mask: batch=%d n_nodes=%d (<= %d)", batch, n_nodes, SA_MAX_NODES);
    if (batch == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!parents || !mask) return ctx_fail(c, DS_CUDA_EINVAL, "tree_mask: null pointer");
    const CtxDevice on(c);
    cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    tree_mask_kernel<<<batch, (n_nodes + 31) & ~31, 0, st>>>(parents, nodes, n_nodes, (n_nodes + 63) / 64, mask, depth);
    return ctx_cuda(c, cudaGetLastError(), "tree_mask launch");
}
