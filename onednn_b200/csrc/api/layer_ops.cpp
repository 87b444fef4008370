// The operators around the matmul of a transformer's layer: fused root-mean-square norm with
// an 8-bit destination, the paged 8-bit cache of keys and values (append, read), and attention
// over it.  Extensions without counterparts in the reference, built like its primitives:
// descriptor checks and dispatch here, one launcher of onednn_b200_kernels.h behind each.
//
// Every execution argument of these primitives has one descriptor, fixed at creation and kept in
// pd->ext_args: that is what dnnl_query_exec_arg_md answers, and what the memories given at
// execution are compared with, so that no kernel sees a tensor other than the one it was
// checked for.
#include <cuda_runtime.h>

#include <cmath>
#include <limits>
#include <new>

#include "internal.hpp"

using namespace b200;

namespace {

bool is_float(int dt) { return dt == dnnl_f32 || dt == dnnl_bf16 || dt == dnnl_f16; }
bool is_code(int dt) { return dt == dnnl_s8 || dt == dnnl_f8_e4m3; }

dnnl_memory_desc dense(int dt, std::initializer_list<int64_t> dims) {
    dnnl_memory_desc md;
    for (int64_t d : dims) md.dims[md.ndims++] = d;
    int64_t s = 1;
    for (int i = md.ndims - 1; i >= 0; --i) {
        md.strides[i] = s;
        s *= std::max<int64_t>(md.dims[i], 1);
    }
    md.data_type = dt;
    md.format_kind = dnnl_blocked;
    return md;
}

// a descriptor these primitives can take: plain, sizes known, contiguous in its last dim (that no
// two elements share a place, its creation has checked)
dnnl_status_t check_plain(const dnnl_memory_desc &md) {
    if (md.ndims < 1) return dnnl_invalid_arguments;
    if (md.is_any() || md.has_runtime_dims() || !md.is_plain()) return dnnl_unimplemented;
    if (md.dims[md.ndims - 1] > 1 && md.strides[md.ndims - 1] != 1) return dnnl_unimplemented;
    return dnnl_success;
}

dnnl_status_t check_attr(const_dnnl_primitive_attr_t attr) {
    if (!attr) return dnnl_success;
    if (!attr->scales.empty() || !attr->zero_points.empty() || !attr->post_ops.entries.empty() || !attr->rounding.empty())
        return dnnl_unimplemented;
    return dnnl_success;
}

// the leading dims of a tensor as rows of one stride
bool fold_rows(const dnnl_memory_desc &md, int64_t &rows, int64_t &stride) {
    rows = 1;
    stride = md.dims[md.ndims - 1];
    for (int i = md.ndims - 2; i >= 0; --i) {
        if (md.dims[i] == 1) continue;
        if (rows == 1) stride = md.strides[i];
        else if (md.strides[i] != stride * rows) return false;
        rows *= md.dims[i];
    }
    return true;
}

using pd_ptr = std::unique_ptr<dnnl_primitive_desc>;

pd_ptr new_pd(dnnl_primitive_kind_t kind, dnnl_engine *engine, const_dnnl_primitive_attr_t attr) {
    pd_ptr pd(new dnnl_primitive_desc());
    pd->kind = kind;
    pd->engine = engine;
    if (attr) pd->attr = *attr;
    return pd;
}

dnnl_status_t finish(pd_ptr &pd, dnnl_primitive_desc_t *out, double t0) {
    pd->user_src = pd->src;
    pd->user_dst = pd->dst;
    pd->engine->refs.fetch_add(1);
    verbose_create(pd.get(), now_ms() - t0, false);
    *out = pd.release();
    return dnnl_success;
}

// rows (tokens, heads, dim) of a ragged batch
dnnl_status_t check_rows(const dnnl_memory_desc &md, int64_t heads, int64_t dim) {
    if (md.ndims != 3) return dnnl_invalid_arguments;
    const dnnl_status_t st = check_plain(md);
    if (st != dnnl_success) return st;
    if (md.dims[2] != dim || (heads && md.dims[1] != heads)) return dnnl_invalid_arguments;
    if (!is_float(md.data_type)) return dnnl_unimplemented;
    if (md.dims[0] > std::numeric_limits<int32_t>::max()) return dnnl_unimplemented; // offsets are s32
    return dnnl_success;
}

dnnl_status_t check_cache(const dnnl_memory_desc &cache, const dnnl_memory_desc &table) {
    if (cache.ndims != 4 || table.ndims != 2) return dnnl_invalid_arguments;
    for (const dnnl_memory_desc *md : {&cache, &table}) {
        const dnnl_status_t st = check_plain(*md);
        if (st != dnnl_success) return st;
    }
    if (!is_code(cache.data_type)) return dnnl_unimplemented;
    if (table.data_type != dnnl_s32) return dnnl_invalid_arguments;
    if (cache.dims[1] < 1 || cache.dims[2] < 1 || cache.dims[3] < 1) return dnnl_invalid_arguments;
    // heads are a grid dimension of the kernels; positions in a sequence are s32
    if (cache.dims[1] > 65535 || table.dims[0] > (1 << 24)) return dnnl_unimplemented;
    // the kernels count inside a page, and across the heads of a token, in 32 bits
    if (cache.dims[2] > (1 << 20) || cache.dims[3] > (1 << 20)) return dnnl_unimplemented;
    if (cache.dims[2] * cache.dims[3] > (1 << 30) || cache.dims[1] * cache.dims[3] > (1 << 30)) return dnnl_unimplemented;
    if (cache.dims[0] > std::numeric_limits<int32_t>::max()) return dnnl_unimplemented; // pages are s32
    return dnnl_success;
}

void cache_args(dnnl_primitive_desc *pd, const dnnl_memory_desc &cache, const dnnl_memory_desc &table) {
    const dnnl_memory_desc scales = dense(dnnl_f32, {cache.dims[0], cache.dims[1]});
    pd->ext_args[DNNL_ARG_B200_KEY_CACHE] = cache;
    pd->ext_args[DNNL_ARG_B200_VALUE_CACHE] = cache;
    pd->ext_args[DNNL_ARG_B200_KEY_SCALES] = scales;
    pd->ext_args[DNNL_ARG_B200_VALUE_SCALES] = scales;
    pd->ext_args[DNNL_ARG_B200_PAGE_TABLE] = table;
    pd->ext_args[DNNL_ARG_B200_SEQ_OFFSETS] = dense(dnnl_s32, {table.dims[0] + 1});
    pd->ext_args[DNNL_ARG_B200_KV_LENS] = dense(dnnl_s32, {table.dims[0]});
}

// where an argument's first element is
void *at(const std::map<int, dnnl_memory *> &args, int arg) {
    auto it = args.find(arg);
    if (it == args.end() || !it->second->handle) return nullptr;
    const dnnl_memory_desc &md = it->second->md;
    return (char *)it->second->handle + md.offset0 * dt_nbits(md.data_type) / 8;
}

// Whether two tensors of one descriptor, `d` elements apart, have an element in common: d is a sum of whole multiples of the
// strides, each of fewer than the dim's size.  Strides are nested (the descriptor's creation has checked), so for each from
// the largest on only the two multiples next to what is left can do.
bool overlap(const dnnl_memory_desc &md, int64_t d, uint32_t done = 0) {
    int big = -1;
    for (int i = 0; i < md.ndims; ++i)
        if (!(done >> i & 1) && md.dims[i] > 1 && (big < 0 || md.strides[i] > md.strides[big])) big = i;
    if (big < 0) return d == 0;
    const int64_t s = md.strides[big], n = md.dims[big], q = d / s - (d % s < 0);
    for (const int64_t k : {q, q + 1})
        if (k > -n && k < n && overlap(md, d - k * s, done | 1u << big)) return true;
    return false;
}
// the same for two arguments; neither empty.  (What begins inside an element of the other's has been refused where elements
// have to be aligned; 8-bit ones always are.)
bool overlap(const std::map<int, dnnl_memory *> &args, int one, int other) {
    const dnnl_memory_desc &md = args.at(one)->md;
    const int64_t bytes = (char *)at(args, other) - (char *)at(args, one);
    return overlap(md, bytes / (dt_nbits(md.data_type) / 8));
}

dnnl_status_t status_of(int rc) {
    if (rc == 0) return dnnl_success;
    if (rc == B200_ERR_UNSUPPORTED || rc == B200_ERR_TOO_LARGE) return dnnl_unimplemented;
    if (rc == B200_ERR_BAD_ARG) return dnnl_invalid_arguments;
    return dnnl_runtime_error;
}

b200_kv_cache_t cache_of(const dnnl_primitive_desc *pd, dnnl_stream *stream, const std::map<int, dnnl_memory *> &args) {
    const dnnl_memory_desc &c = pd->ext_args.at(DNNL_ARG_B200_KEY_CACHE), &t = pd->ext_args.at(DNNL_ARG_B200_PAGE_TABLE);
    b200_kv_cache_t k;
    std::memset(&k, 0, sizeof(k));
    k.key = at(args, DNNL_ARG_B200_KEY_CACHE);
    k.value = at(args, DNNL_ARG_B200_VALUE_CACHE);
    k.key_scale = (float *)at(args, DNNL_ARG_B200_KEY_SCALES);
    k.value_scale = (float *)at(args, DNNL_ARG_B200_VALUE_SCALES);
    k.dt = c.data_type;
    k.pages = c.dims[0];
    k.heads = c.dims[1];
    k.page = c.dims[2];
    k.dim = c.dims[3];
    k.s_page = c.strides[0];
    k.s_head = c.strides[1];
    k.s_slot = c.strides[2];
    k.table = (const int32_t *)at(args, DNNL_ARG_B200_PAGE_TABLE);
    k.table_s0 = t.strides[0];
    k.table_cols = t.dims[1];
    k.offsets = (const int32_t *)at(args, DNNL_ARG_B200_SEQ_OFFSETS);
    k.lens = (const int32_t *)at(args, DNNL_ARG_B200_KV_LENS);
    k.seqs = t.dims[0];
    k.status = stream->status;
    return k;
}

dnnl_status_t norm_execute(const dnnl_primitive_desc *pd, dnnl_stream *stream, const std::map<int, dnnl_memory *> &args) {
    b200_rms_norm_params_t p;
    std::memset(&p, 0, sizeof(p));
    int64_t rows;
    p.cols = pd->src.dims[pd->src.ndims - 1];
    (void)fold_rows(pd->src, p.rows, p.src_s0);
    (void)fold_rows(pd->dst, rows, p.dst_s0);
    p.src = at(args, DNNL_ARG_SRC);
    p.src_dt = pd->src.data_type;
    p.dst = at(args, DNNL_ARG_DST);
    p.dst_dt = pd->dst.data_type;
    auto res = pd->ext_args.find(DNNL_ARG_SRC_1);
    if (res != pd->ext_args.end()) {
        (void)fold_rows(res->second, rows, p.residual_s0);
        p.sum_s0 = p.residual_s0;
        p.residual = at(args, DNNL_ARG_SRC_1);
        p.sum = at(args, DNNL_ARG_DST_1);
        p.residual_dt = res->second.data_type;
    }
    auto gamma = pd->ext_args.find(DNNL_ARG_SCALE);
    if (gamma != pd->ext_args.end()) {
        p.gamma = at(args, DNNL_ARG_SCALE);
        p.gamma_dt = gamma->second.data_type;
    }
    p.row_scale = (float *)at(args, DNNL_ARG_ATTR_SCALES | DNNL_ARG_DST);
    p.epsilon = pd->ext_param;
    return status_of(b200_rms_norm_launch(&p, stream->cuda_stream));
}

dnnl_status_t kv_rows_execute(const dnnl_primitive_desc *pd, dnnl_stream *stream, const std::map<int, dnnl_memory *> &args) {
    const bool append = pd->kind == dnnl_b200_kv_cache_append;
    const dnnl_memory_desc &rows = append ? pd->src : pd->dst;
    b200_kv_rows_params_t p;
    std::memset(&p, 0, sizeof(p));
    p.cache = cache_of(pd, stream, args);
    p.key = at(args, append ? DNNL_ARG_SRC : DNNL_ARG_DST);
    p.value = at(args, append ? DNNL_ARG_SRC_1 : DNNL_ARG_DST_1);
    p.dt = rows.data_type;
    p.rows = rows.dims[0];
    p.s_row = rows.strides[0];
    p.s_head = rows.strides[1];
    return status_of(append ? b200_kv_append_launch(&p, stream->cuda_stream) : b200_kv_read_launch(&p, stream->cuda_stream));
}

// The attention implementations of this engine, in dispatch order.
struct attention_impl_t {
    const char *name;
    int (*supported)(const b200_kv_attention_params_t *);
    size_t (*scratch_bytes)(const b200_kv_attention_params_t *);
    int (*launch)(const b200_kv_attention_params_t *, b200_stream_t);
};
const attention_impl_t attention_impls[] = {
        {"cuda:sm100:kv_attention_tc", b200_kv_attention_tc_supported, b200_kv_attention_tc_scratch_bytes,
                b200_kv_attention_tc_launch},
        {"cuda:sm100:kv_attention_mma", b200_kv_attention_mma_supported, b200_kv_attention_mma_scratch_bytes,
                b200_kv_attention_mma_launch},
        {"cuda:generic", nullptr, nullptr, b200_kv_attention_generic_launch}};
constexpr int ATTENTION_IMPLS = sizeof(attention_impls) / sizeof(attention_impls[0]);

// what the descriptors say; the pointers stay NULL
b200_kv_attention_params_t attention_params(const dnnl_primitive_desc *pd) {
    b200_kv_attention_params_t p;
    std::memset(&p, 0, sizeof(p));
    const dnnl_memory_desc &c = pd->ext_args.at(DNNL_ARG_B200_KEY_CACHE), &t = pd->ext_args.at(DNNL_ARG_B200_PAGE_TABLE);
    p.cache.dt = c.data_type;
    p.cache.pages = c.dims[0];
    p.cache.heads = c.dims[1];
    p.cache.page = c.dims[2];
    p.cache.dim = c.dims[3];
    p.cache.s_page = c.strides[0];
    p.cache.s_head = c.strides[1];
    p.cache.s_slot = c.strides[2];
    p.cache.seqs = t.dims[0];
    p.cache.table_s0 = t.strides[0];
    p.cache.table_cols = t.dims[1];
    p.query_dt = pd->src.data_type;
    p.query_s0 = pd->src.strides[0];
    p.query_s1 = pd->src.strides[1];
    p.dst_dt = pd->dst.data_type;
    p.dst_s0 = pd->dst.strides[0];
    p.dst_s1 = pd->dst.strides[1];
    p.rows = pd->src.dims[0];
    p.q_heads = pd->src.dims[1];
    p.scale = pd->ext_param;
    p.sm_count = pd->engine->sm_count;
    return p;
}

// the first implementation from `first` on that takes the problem
dnnl_status_t attention_select(dnnl_primitive_desc *pd, int first) {
    b200_kv_attention_params_t p = attention_params(pd);
    // offset0 moves where the first element is: a pointer of that value stands for it
    const auto place = [](const dnnl_memory_desc &md) { return (char *)nullptr + md.offset0 * dt_nbits(md.data_type) / 8; };
    p.query = place(pd->src);
    p.dst = place(pd->dst);
    p.cache.key = p.cache.value = place(pd->ext_args.at(DNNL_ARG_B200_KEY_CACHE));
    for (int i = first; i < ATTENTION_IMPLS; ++i) {
        const attention_impl_t &impl = attention_impls[i];
        if (impl.supported && !impl.supported(&p)) continue;
        pd->impl = i;
        pd->impl_str = impl.name;
        pd->scratchpad = dnnl_memory_desc();
        // sizes only; a descriptor-only engine has no multiprocessors, and nothing to run on
        const size_t bytes = impl.scratch_bytes ? impl.scratch_bytes(&p) : 0;
        if (bytes) pd->scratchpad = dense(dnnl_u8, {(int64_t)bytes});
        return dnnl_success;
    }
    return dnnl_unimplemented;
}

dnnl_status_t attention_execute(const dnnl_primitive *prim, dnnl_stream *stream, const std::map<int, dnnl_memory *> &args) {
    const dnnl_primitive_desc *pd = prim->pd.get();
    b200_kv_attention_params_t p = attention_params(pd);
    p.cache = cache_of(pd, stream, args);
    p.query = at(args, DNNL_ARG_SRC);
    p.dst = at(args, DNNL_ARG_DST);
    const attention_impl_t *impl = &attention_impls[pd->impl];
    // buffers that start where 16-byte accesses cannot (the descriptors' strides were checked at creation)
    if (impl->supported && !impl->supported(&p)) impl = &attention_impls[ATTENTION_IMPLS - 1];
    p.scratch_bytes = impl->scratch_bytes && pd->scratchpad.ndims ? (size_t)pd->scratchpad.dims[0] : 0;
    if (!p.scratch_bytes) return status_of(impl->launch(&p, stream->cuda_stream));

    const cudaStream_t cs = (cudaStream_t)stream->cuda_stream;
    if (pd->attr.scratchpad_mode == dnnl_scratchpad_mode_user) {
        auto it = args.find(DNNL_ARG_SCRATCHPAD);
        if (it == args.end() || !it->second->handle || it->second->md.size_bytes() < p.scratch_bytes) return dnnl_invalid_arguments;
        p.scratch = at(args, DNNL_ARG_SCRATCHPAD);
        if ((uintptr_t)p.scratch % 16 != 0) return dnnl_invalid_arguments; // partial results are read 16 bytes at a time
        return status_of(impl->launch(&p, cs));
    }
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(cs, &capture) != cudaSuccess) {
        (void)cudaGetLastError();
        return dnnl_runtime_error;
    }
    if (capture != cudaStreamCaptureStatusNone) {
        // a graph may be replayed next to others and to eager executions: it gets memory of its own
        if (device_alloc_async(&p.scratch, p.scratch_bytes, cs) != cudaSuccess) {
            (void)cudaGetLastError();
            return dnnl_out_of_memory;
        }
        const dnnl_status_t st = status_of(impl->launch(&p, cs));
        if (cudaFreeAsync(p.scratch, cs) != cudaSuccess) return dnnl_runtime_error;
        return st;
    }
    // as for the matmul: zeroed at creation, left zeroed, cleared again after an error
    p.scratch = prim->lib_scratch;
    if (!p.scratch) return dnnl_out_of_memory;
    const uint64_t now = g_scratch_epoch.load();
    if (prim->scratch_epoch.exchange(now) == now) p.scratch_zeroed = 1;
    else g_scratch_reclears.fetch_add(1);
    return status_of(impl->launch(&p, cs));
}

} // namespace

namespace b200 {

bool is_ext_kind(int kind) { return kind >= dnnl_b200_rms_norm && kind <= dnnl_b200_kv_cache_attention; }

const char *ext_kind_name(int kind) {
    switch (kind) {
        case dnnl_b200_rms_norm: return "b200_rms_norm";
        case dnnl_b200_kv_cache_append: return "b200_kv_cache_append";
        case dnnl_b200_kv_cache_read: return "b200_kv_cache_read";
        default: return "b200_kv_cache_attention";
    }
}

dnnl_status_t ext_next_impl(dnnl_primitive_desc *pd) {
    if (pd->kind != dnnl_b200_kv_cache_attention) return dnnl_last_impl_reached; // one implementation
    return attention_select(pd, pd->impl + 1) == dnnl_success ? dnnl_success : dnnl_last_impl_reached;
}

dnnl_status_t ext_execute(const dnnl_primitive *prim, dnnl_stream *stream, const std::map<int, dnnl_memory *> &args) {
    const dnnl_primitive_desc *pd = prim->pd.get();
    const dnnl_memory_desc &rows = pd->kind == dnnl_b200_kv_cache_read ? pd->dst : pd->src;
    if (rows.has_zero_dim()) return dnnl_success;
    for (const auto &want : pd->ext_args) {
        auto it = args.find(want.first);
        if (it == args.end() || !it->second->md.equal(want.second)) return dnnl_invalid_arguments;
        if (!it->second->handle && !want.second.has_zero_dim()) return dnnl_invalid_arguments;
        // no element may straddle its type's boundary: a kernel that read it would fault
        if ((uintptr_t)it->second->handle % (dt_nbits(want.second.data_type) / 8) != 0) return dnnl_invalid_arguments;
    }
    // keys and values are written side by side: in places that they share they would race
    if (pd->kind == dnnl_b200_kv_cache_append && !pd->dst.has_zero_dim()
            && (overlap(args, DNNL_ARG_B200_KEY_SCALES, DNNL_ARG_B200_VALUE_SCALES)
                    || overlap(args, DNNL_ARG_B200_KEY_CACHE, DNNL_ARG_B200_VALUE_CACHE)))
        return dnnl_invalid_arguments;
    if (pd->kind == dnnl_b200_kv_cache_read && overlap(args, DNNL_ARG_DST, DNNL_ARG_DST_1)) return dnnl_invalid_arguments;
    // and a row's result would be written over its sum
    if (pd->kind == dnnl_b200_rms_norm && pd->ext_args.count(DNNL_ARG_DST_1) && at(args, DNNL_ARG_DST) == at(args, DNNL_ARG_DST_1))
        return dnnl_invalid_arguments;
    switch (pd->kind) {
        case dnnl_b200_rms_norm: return norm_execute(pd, stream, args);
        case dnnl_b200_kv_cache_attention: return attention_execute(prim, stream, args);
        default: return kv_rows_execute(pd, stream, args);
    }
}

} // namespace b200

dnnl_status_t dnnl_b200_rms_norm_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t residual_desc, const_dnnl_memory_desc_t scale_desc,
        const_dnnl_memory_desc_t dst_desc, float epsilon, const_dnnl_primitive_attr_t attr) try {
    if (!primitive_desc || !engine || !src_desc || !dst_desc) return dnnl_invalid_arguments;
    const double t0 = now_ms();
    if (!(epsilon >= 0.f) || std::isinf(epsilon)) return dnnl_invalid_arguments;
    if (engine->host) return dnnl_unimplemented;
    dnnl_status_t st = check_attr(attr);
    if (st != dnnl_success) return st;
    for (const dnnl_memory_desc *md : {src_desc, residual_desc, dst_desc}) {
        if (!md) continue;
        if ((st = check_plain(*md)) != dnnl_success) return st;
        if (md->ndims != src_desc->ndims) return dnnl_invalid_arguments;
        for (int i = 0; i < md->ndims; ++i)
            if (md->dims[i] != src_desc->dims[i]) return dnnl_invalid_arguments;
        int64_t rows, stride;
        if (!fold_rows(*md, rows, stride)) return dnnl_unimplemented;
        if (rows > std::numeric_limits<int32_t>::max()) return dnnl_unimplemented; // rows are a grid dimension
    }
    if (src_desc->dims[src_desc->ndims - 1] > std::numeric_limits<int32_t>::max()) return dnnl_unimplemented;
    if (!is_float(src_desc->data_type) || (residual_desc && !is_float(residual_desc->data_type))) return dnnl_unimplemented;
    if (!is_float(dst_desc->data_type) && !is_code(dst_desc->data_type)) return dnnl_unimplemented;
    if (scale_desc) {
        if (scale_desc->ndims != 1 || scale_desc->dims[0] != src_desc->dims[src_desc->ndims - 1]) return dnnl_invalid_arguments;
        if ((st = check_plain(*scale_desc)) != dnnl_success) return st;
        if (!is_float(scale_desc->data_type)) return dnnl_unimplemented;
    }
    pd_ptr pd = new_pd(dnnl_b200_rms_norm, engine, attr);
    pd->src = *src_desc;
    pd->dst = *dst_desc;
    pd->ext_param = epsilon;
    pd->ext_args[DNNL_ARG_SRC] = *src_desc;
    pd->ext_args[DNNL_ARG_DST] = *dst_desc;
    pd->ext_inputs = pd->ext_outputs = 1;
    if (residual_desc) {
        pd->ext_args[DNNL_ARG_SRC_1] = *residual_desc;
        pd->ext_args[DNNL_ARG_DST_1] = *residual_desc;
        ++pd->ext_inputs;
        ++pd->ext_outputs;
    }
    if (scale_desc) {
        pd->ext_args[DNNL_ARG_SCALE] = *scale_desc;
        ++pd->ext_inputs;
    }
    if (is_code(dst_desc->data_type)) {
        int64_t rows, stride;
        (void)fold_rows(*dst_desc, rows, stride);
        pd->ext_args[DNNL_ARG_ATTR_SCALES | DNNL_ARG_DST] = dense(dnnl_f32, {rows});
        ++pd->ext_outputs;
    }
    pd->impl = 0;
    pd->impl_str = "cuda:rms_norm";
    return finish(pd, primitive_desc, t0);
} catch (const std::bad_alloc &) { return dnnl_out_of_memory; }

dnnl_status_t dnnl_b200_kv_cache_append_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t src_desc, const_dnnl_memory_desc_t cache_desc, const_dnnl_memory_desc_t table_desc,
        const_dnnl_primitive_attr_t attr) try {
    if (!primitive_desc || !engine || !src_desc || !cache_desc || !table_desc) return dnnl_invalid_arguments;
    const double t0 = now_ms();
    if (engine->host) return dnnl_unimplemented;
    dnnl_status_t st = check_attr(attr);
    if (st == dnnl_success) st = check_cache(*cache_desc, *table_desc);
    if (st == dnnl_success) st = check_rows(*src_desc, cache_desc->dims[1], cache_desc->dims[3]);
    if (st != dnnl_success) return st;
    pd_ptr pd = new_pd(dnnl_b200_kv_cache_append, engine, attr);
    pd->src = *src_desc;
    pd->dst = *cache_desc;
    cache_args(pd.get(), *cache_desc, *table_desc);
    pd->ext_args[DNNL_ARG_SRC] = pd->ext_args[DNNL_ARG_SRC_1] = *src_desc;
    pd->ext_inputs = 5;
    pd->ext_outputs = 4;
    pd->impl = 0;
    pd->impl_str = "cuda:kv_append";
    return finish(pd, primitive_desc, t0);
} catch (const std::bad_alloc &) { return dnnl_out_of_memory; }

dnnl_status_t dnnl_b200_kv_cache_read_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t cache_desc, const_dnnl_memory_desc_t dst_desc, const_dnnl_memory_desc_t table_desc,
        const_dnnl_primitive_attr_t attr) try {
    if (!primitive_desc || !engine || !cache_desc || !dst_desc || !table_desc) return dnnl_invalid_arguments;
    const double t0 = now_ms();
    if (engine->host) return dnnl_unimplemented;
    dnnl_status_t st = check_attr(attr);
    if (st == dnnl_success) st = check_cache(*cache_desc, *table_desc);
    if (st == dnnl_success) st = check_rows(*dst_desc, cache_desc->dims[1], cache_desc->dims[3]);
    if (st != dnnl_success) return st;
    pd_ptr pd = new_pd(dnnl_b200_kv_cache_read, engine, attr);
    pd->src = *cache_desc;
    pd->dst = *dst_desc;
    cache_args(pd.get(), *cache_desc, *table_desc);
    pd->ext_args[DNNL_ARG_DST] = pd->ext_args[DNNL_ARG_DST_1] = *dst_desc;
    pd->ext_inputs = 7;
    pd->ext_outputs = 2;
    pd->impl = 0;
    pd->impl_str = "cuda:kv_read";
    return finish(pd, primitive_desc, t0);
} catch (const std::bad_alloc &) { return dnnl_out_of_memory; }

dnnl_status_t dnnl_b200_kv_cache_attention_primitive_desc_create(dnnl_primitive_desc_t *primitive_desc, dnnl_engine_t engine,
        const_dnnl_memory_desc_t query_desc, const_dnnl_memory_desc_t cache_desc, const_dnnl_memory_desc_t dst_desc,
        const_dnnl_memory_desc_t table_desc, float softmax_scale, const_dnnl_primitive_attr_t attr) try {
    if (!primitive_desc || !engine || !query_desc || !cache_desc || !dst_desc || !table_desc) return dnnl_invalid_arguments;
    const double t0 = now_ms();
    if (!std::isfinite(softmax_scale)) return dnnl_invalid_arguments;
    if (engine->host) return dnnl_unimplemented;
    dnnl_status_t st = check_attr(attr);
    if (st == dnnl_success) st = check_cache(*cache_desc, *table_desc);
    for (const dnnl_memory_desc *md : {query_desc, dst_desc})
        if (st == dnnl_success) st = check_rows(*md, 0, cache_desc->dims[3]);
    if (st != dnnl_success) return st;
    if (query_desc->dims[0] != dst_desc->dims[0] || query_desc->dims[1] != dst_desc->dims[1]) return dnnl_invalid_arguments;
    if (query_desc->dims[1] < 1 || query_desc->dims[1] % cache_desc->dims[1] != 0) return dnnl_invalid_arguments;
    if (cache_desc->dims[3] > 256 || query_desc->dims[1] > 65535) return dnnl_unimplemented;
    // query rows of a key head are counted in 32 bits
    if (query_desc->dims[0] * (query_desc->dims[1] / cache_desc->dims[1]) > 0x7fffff00) return dnnl_unimplemented;
    pd_ptr pd = new_pd(dnnl_b200_kv_cache_attention, engine, attr);
    pd->src = *query_desc;
    pd->dst = *dst_desc;
    pd->ext_param = softmax_scale;
    cache_args(pd.get(), *cache_desc, *table_desc);
    pd->ext_args[DNNL_ARG_SRC] = *query_desc;
    pd->ext_args[DNNL_ARG_DST] = *dst_desc;
    pd->ext_inputs = 8;
    pd->ext_outputs = 1;
    if ((st = attention_select(pd.get(), 0)) != dnnl_success) return st;
    return finish(pd, primitive_desc, t0);
} catch (const std::bad_alloc &) { return dnnl_out_of_memory; }
