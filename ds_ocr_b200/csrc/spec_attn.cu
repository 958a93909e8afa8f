// spec_attn.cu — attention of a tree of drafted tokens over the KV cache
// (ds_cuda_tree_attention_dev), and the trees' mask words.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ctx.h"

namespace ds {

constexpr int SA_MAX_NODES = 256;

struct SaArgs {
    ds_cuda_tree_attention_t d;
    int words;  // mask words per node
};

__device__ __forceinline__ float sa_load(const void *p, int64_t i, int type) {
    if (type == DS_CUDA_SPEC_F16) return __half2float(reinterpret_cast<const __half *>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
}

// One CTA per (node, head, sequence): four warps take the keys in turn, each
// lane HD / 32 dimensions, with a running maximum and sum per warp; the
// warps' parts are joined at the end.
template <int HD>
__global__ void __launch_bounds__(128) sa_rows_kernel(const __grid_constant__ SaArgs a) {
    constexpr int PL = HD / 32;
    const ds_cuda_tree_attention_t &d = a.d;
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = h / (d.n_heads / d.n_kv_heads);
    const int len = min(max(d.lens[b], 0), d.kv_max);
    const int cnt = d.nodes ? min(max(d.nodes[b], 0), d.n_nodes) : d.n_nodes;
    const int total = i < cnt ? len + cnt : 0;
    const uint64_t *mask = d.mask + ((size_t)b * d.n_nodes + i) * a.words;
    const int64_t qo = b * d.q_stride[0] + i * d.q_stride[1] + h * d.q_stride[2] + lane * PL;
    float q[PL], o[PL], m = -__FLT_MAX__, l = 0.f;
#pragma unroll
    for (int c = 0; c < PL; c++) {
        q[c] = d.type == DS_CUDA_SPEC_F32 ? reinterpret_cast<const float *>(d.q)[qo + c] : sa_load(d.q, qo + c, d.type);
        q[c] *= d.scale;
        o[c] = 0.f;
    }
    for (int j = warp; j < total; j += 4) {
        const bool node = j >= len;
        const int t = j - len;
        if (node && !((mask[t >> 6] >> (t & 63)) & 1)) continue;
        const void *kp = node ? d.tree_k : d.k, *kl = node ? d.tree_k_lo : d.k_lo;
        const void *vp = node ? d.tree_v : d.v, *vl = node ? d.tree_v_lo : d.v_lo;
        const int64_t *ks = node ? d.tree_k_stride : d.k_stride, *vs = node ? d.tree_v_stride : d.v_stride;
        const int64_t row = node ? t : j;
        const int64_t ko = b * ks[0] + g * ks[1] + row * ks[2] + lane * PL;
        const int64_t vo = b * vs[0] + g * vs[1] + row * vs[2] + lane * PL;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < PL; c++) {
            float k = sa_load(kp, ko + c, d.type);
            if (d.type == DS_CUDA_SPEC_F32 && kl) k += sa_load(kl, ko + c, d.type);
            s += q[c] * k;
        }
        s = warp_sum(s);
        const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
        l = l * f + p;
        m = mn;
#pragma unroll
        for (int c = 0; c < PL; c++) {
            float v = sa_load(vp, vo + c, d.type);
            if (d.type == DS_CUDA_SPEC_F32 && vl) v += sa_load(vl, vo + c, d.type);
            o[c] = o[c] * f + p * v;
        }
    }
    __shared__ float sm[4], sl[4], so[4][HD];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int c = 0; c < PL; c++) so[warp][lane * PL + c] = o[c];
    __syncthreads();
    if (warp) return;
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    l = 0.f;
#pragma unroll
    for (int c = 0; c < PL; c++) o[c] = 0.f;
    for (int w = 0; w < 4; w++) {
        const float f = expf(sm[w] - m);
        l += sl[w] * f;
#pragma unroll
        for (int c = 0; c < PL; c++) o[c] += so[w][lane * PL + c] * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t oo = b * d.out_stride[0] + i * d.out_stride[1] + h * d.out_stride[2] + lane * PL;
#pragma unroll
    for (int c = 0; c < PL; c++) {
        const float x = l == 0.f ? 0.f : o[c] * inv;
        if (d.type == DS_CUDA_SPEC_F32) reinterpret_cast<float *>(d.out)[oo + c] = x;
        else if (d.type == DS_CUDA_SPEC_F16) reinterpret_cast<__half *>(d.out)[oo + c] = __float2half_rn(x);
        else reinterpret_cast<__nv_bfloat16 *>(d.out)[oo + c] = __float2bfloat16_rn(x);
    }
    if (d.lse && lane == 0)
        d.lse[((size_t)b * d.n_nodes + i) * d.n_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

// One CTA per sequence, one thread per node: a node's word bits are set by
// walking up its parents (kept in shared memory; at most n_nodes steps).
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
        d->n_heads % d->n_kv_heads || (d->head_dim != 64 && d->head_dim != 128) || d->kv_max < 0)
        return ctx_fail(c, DS_CUDA_EINVAL,
                        "tree_attention: unsupported shape batch=%d n_nodes=%d n_heads=%d n_kv_heads=%d head_dim=%d "
                        "kv_max=%d (n_nodes <= %d, head_dim 64 or 128, n_heads a multiple of n_kv_heads)",
                        d->batch, d->n_nodes, d->n_heads, d->n_kv_heads, d->head_dim, d->kv_max, SA_MAX_NODES);
    if (d->batch > 65535 || d->n_heads > 65535)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_attention: batch and n_heads are at most 65535");
    return DS_CUDA_OK;
}

extern "C" size_t ds_cuda_tree_attention_workspace(const ds_cuda_ctx_t *c, const ds_cuda_tree_attention_t *d) {
    if (!c || !c->ok || sa_check(nullptr, d) < 0) return 0;
    return 0;
}

extern "C" int ds_cuda_tree_attention_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_attention_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    int rc = sa_check(c, d);
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
    SaArgs a = {*d, (d->n_nodes + 63) / 64};
    cudaSetDevice(c->device);
    cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    const dim3 grid(d->n_nodes, d->n_heads, d->batch);
    if (d->head_dim == 64) sa_rows_kernel<64><<<grid, 128, 0, st>>>(a);
    else sa_rows_kernel<128><<<grid, 128, 0, st>>>(a);
    return ctx_cuda(c, cudaGetLastError(), "tree_attention launch");
}

extern "C" int ds_cuda_tree_mask_dev(ds_cuda_ctx_t *c, const int *parents, const int *nodes, int batch, int n_nodes,
                                     uint64_t *mask, int *depth, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (batch < 0 || n_nodes <= 0 || n_nodes > SA_MAX_NODES)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_mask: batch=%d n_nodes=%d (<= %d)", batch, n_nodes, SA_MAX_NODES);
    if (batch == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!parents || !mask) return ctx_fail(c, DS_CUDA_EINVAL, "tree_mask: null pointer");
    cudaSetDevice(c->device);
    cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    tree_mask_kernel<<<batch, (n_nodes + 31) & ~31, 0, st>>>(parents, nodes, n_nodes, (n_nodes + 63) / 64, mask, depth);
    return ctx_cuda(c, cudaGetLastError(), "tree_mask launch");
}
