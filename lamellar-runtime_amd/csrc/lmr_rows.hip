// lmr_rows.hip — batched load / add / store of whole rows: the records of a batch are rows of a
// table (row_len elements each) instead of single elements.
//
//   lmr_rows_load    out[t, :] = rnd(scale * table[i[t], :])            (an embedding lookup; an
//                    8-bit cache read back: element = code * scale of its group)
//   lmr_rows_add     table[r, :] = rnd(table[r, :] + scale * sum of vals[t, :] over i[t] = r)
//                    (the lookup's gradient; every collision counted, in a fixed order)
//   lmr_rows_store   table[i[t], :] = rnd(vals[t, :]), the last record of a row wins; 8-bit tables
//                    take codes and one f32 scale per group, both of the same record
//
// Arithmetic is f32; each result is rounded once, to the nearest even, when it is written.
#include "lmr_internal.hpp"
#include "lmr_rows.hpp"

namespace lmr {
namespace {

template <int IW>
__device__ __forceinline__ int64_t row_index(const RowBatch& b, uint64_t t) {
    if constexpr (IW == 4) return reinterpret_cast<const int32_t*>(b.idx)[t];
    else return reinterpret_cast<const int64_t*>(b.idx)[t];
}

// the record's row, or -1: a pad, or out of bounds (reported by `lead` threads)
template <int IW>
__device__ __forceinline__ int64_t row_of(const RowBatch& b, uint64_t t, uint64_t rows, uint32_t* err, bool lead) {
    const int64_t i = row_index<IW>(b, t);
    if (b.has_pad && i == b.pad) return -1;
    if (uint64_t(i) >= rows) {
        if (lead) atomicOr(err, LMR_ERRBIT_OOB);
        return -1;
    }
    return i;
}

// one block per record
template <typename T, typename O, int IW>
__global__ __launch_bounds__(256) void k_rows_load(RowTable tab, RowBatch b, O* out, uint32_t* err) {
    const uint64_t t = blockIdx.x;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, threadIdx.x == 0);
    for (uint64_t j = threadIdx.x; j < tab.row_len; j += blockDim.x) {
        float v = 0.f;
        if (r >= 0) {
            v = to_f32(reinterpret_cast<const T*>(tab.data)[uint64_t(r) * tab.row_len + j]);
            if constexpr (is_code<T>::v) v *= tab.scales[uint64_t(r) * tab.groups + j / tab.group];
            v *= b.scale;
        }
        out[t * b.stride + j] = from_f32<O>(v);
    }
}

// one block per record: the first record of a row sums the row's records in order
template <typename T, typename V, int IW>
__global__ __launch_bounds__(256) void k_rows_add(RowTable tab, RowBatch b, const V* vals, uint32_t* err) {
    const uint64_t t = blockIdx.x;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, threadIdx.x == 0);
    if (r < 0) return;
    bool earlier = false;
    for (uint64_t u = threadIdx.x & 63; u < t; u += 64) earlier |= row_index<IW>(b, u) == r;
    if (__ballot(earlier)) return;                       // (every wave of the block votes alike)
    T* row = reinterpret_cast<T*>(tab.data) + uint64_t(r) * tab.row_len;
    for (uint64_t j = threadIdx.x; j < tab.row_len; j += blockDim.x) {
        float acc = 0.f;
        for (uint64_t u = t; u < b.n; u++)
            if (row_index<IW>(b, u) == r) acc += to_f32(vals[u * b.stride + j]);
        row[j] = from_f32<T>(fmaf(b.scale, acc, to_f32(row[j])));
    }
}

// one block per record; a record that a later one overwrites does nothing
template <typename T, typename V, int IW>
__global__ __launch_bounds__(64) void k_rows_store(RowTable tab, RowBatch b, const V* vals, uint32_t* err) {
    const uint64_t t = blockIdx.x;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, threadIdx.x == 0);
    if (r < 0) return;
    bool later = false;
    if (tab.claims)
        for (uint64_t u = t + 1 + threadIdx.x; u < b.n; u += 64) later |= row_index<IW>(b, u) == r;
    if (__ballot(later)) return;
    T* row = reinterpret_cast<T*>(tab.data) + uint64_t(r) * tab.row_len;
    const V* x = vals + t * b.stride;
    if constexpr (!is_code<T>::v) {
        for (uint64_t j = threadIdx.x; j < tab.row_len; j += 64) row[j] = from_f32<T>(to_f32(x[j]));
    } else {
        for (uint64_t g = 0; g < tab.groups; g++) {
            uint32_t m = 0;                              // largest |x| as bits: infinities and NaN above every number
            for (uint64_t j = threadIdx.x; j < tab.group; j += 64)
                m = max(m, __float_as_uint(to_f32(x[g * tab.group + j])) & 0x7fffffffu);
            for (int d = 32; d; d >>= 1) m = max(m, uint32_t(__shfl_xor(int(m), d, 64)));
            const GroupScale q = group_scale<T>(m);
            for (uint64_t j = threadIdx.x; j < tab.group; j += 64)
                row[g * tab.group + j] = to_code<T>(to_f32(x[g * tab.group + j]), q);
            if (threadIdx.x == 0) tab.scales[uint64_t(r) * tab.groups + g] = q.scale;
        }
    }
}

template <typename F>
hipError_t by_value_type(uint32_t type, F&& f) {
    switch (type) {
    case LMR_ROW_F32: return f(float{});
    case LMR_ROW_F16: return f(_Float16{});
    default: return f(__bf16{});
    }
}
template <typename F>
hipError_t by_row_type(uint32_t type, F&& f) {
    switch (type) {
    case LMR_ROW_I8: return f(code_i8{});
    case LMR_ROW_E4M3: return f(code_e4m3{});
    default: return by_value_type(type, f);
    }
}
template <typename F>
hipError_t by_index(uint32_t size, F&& f) {
    return size == 4 ? f(std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 8>{});
}

hipError_t launch_load(const RowTable& tab, const RowBatch& b, void* out, uint32_t out_type, uint32_t* err, hipStream_t s) {
    return by_row_type(tab.type, [&](auto t) { return by_value_type(out_type, [&](auto o) { return by_index(b.index_size, [&](auto iw) {
        hipLaunchKernelGGL((k_rows_load<decltype(t), decltype(o), decltype(iw)::value>), dim3(unsigned(b.n)), dim3(256), 0, s,
                           tab, b, reinterpret_cast<decltype(o)*>(out), err);
        return hipGetLastError();
    }); }); });
}
hipError_t launch_add(const RowTable& tab, const RowBatch& b, const void* vals, uint32_t val_type, uint32_t* err, hipStream_t s) {
    return by_value_type(tab.type, [&](auto t) { return by_value_type(val_type, [&](auto v) { return by_index(b.index_size, [&](auto iw) {
        hipLaunchKernelGGL((k_rows_add<decltype(t), decltype(v), decltype(iw)::value>), dim3(unsigned(b.n)), dim3(256), 0, s,
                           tab, b, reinterpret_cast<const decltype(v)*>(vals), err);
        return hipGetLastError();
    }); }); });
}
hipError_t launch_store(const RowTable& tab, const RowBatch& b, const void* vals, uint32_t val_type, uint32_t* err, hipStream_t s) {
    return by_row_type(tab.type, [&](auto t) { return by_value_type(val_type, [&](auto v) { return by_index(b.index_size, [&](auto iw) {
        hipLaunchKernelGGL((k_rows_store<decltype(t), decltype(v), decltype(iw)::value>), dim3(unsigned(b.n)), dim3(64), 0, s,
                           tab, b, reinterpret_cast<const decltype(v)*>(vals), err);
        return hipGetLastError();
    }); }); });
}

uint32_t type_bytes(uint32_t type) {
    switch (type) {
    case LMR_ROW_F32: return 4;
    case LMR_ROW_F16: case LMR_ROW_BF16: return 2;
    default: return 1;
    }
}
bool aligned(const void* p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

lmr_status_t check_table(const lmr_rows_t* t) {
    if (!t || t->type >= LMR_NUM_ROW_TYPES) return LMR_E_INVALID;
    if (t->row_len == 0 || t->row_len > LMR_ROW_MAX_LEN || t->rows > LMR_ROWS_MAX) return LMR_E_INVALID;
    if (t->rows && (!t->data || !aligned(t->data, type_bytes(t->type)))) return LMR_E_INVALID;
    if (t->claims && !aligned(t->claims, 4)) return LMR_E_INVALID;
    if (t->type == LMR_ROW_I8 || t->type == LMR_ROW_E4M3) {
        if (t->group == 0 || t->row_len % t->group != 0) return LMR_E_INVALID;
        if (t->rows && (!t->scales || !aligned(t->scales, 4))) return LMR_E_INVALID;
    }
    return LMR_OK;
}

// the records and the n x row_len values beside them (load: the output; stride 0: one row for every record)
lmr_status_t check_batch(const lmr_ctx* ctx, const lmr_rows_t* t, const void* idx, uint32_t index_size, uint64_t n,
                         const void* vals, uint32_t val_type, uint64_t stride, bool may_repeat) {
    if (!ctx) return LMR_E_INVALID;
    const lmr_status_t st = check_table(t);
    if (st != LMR_OK) return st;
    if ((index_size != 4 && index_size != 8) || val_type > LMR_ROW_BF16 || n > LMR_ROW_MAX_BATCH) return LMR_E_INVALID;
    if (n > 0 && (!idx || !vals || !aligned(idx, index_size) || !aligned(vals, type_bytes(val_type)))) return LMR_E_INVALID;
    if (n > 1 && stride < t->row_len && !(may_repeat && stride == 0)) return LMR_E_INVALID;
    if (stride > (uint64_t(1) << 40)) return LMR_E_INVALID;
    return LMR_OK;
}

RowTable table_of(const lmr_rows_t* t) {
    RowTable r;
    r.data = t->data;
    r.scales = t->scales;
    r.claims = t->claims;
    r.rows = t->rows;
    r.row_len = uint32_t(t->row_len);
    r.type = t->type;
    const bool code = t->type == LMR_ROW_I8 || t->type == LMR_ROW_E4M3;
    r.group = code ? t->group : uint32_t(t->row_len);
    r.groups = uint32_t(t->row_len) / r.group;
    return r;
}
RowBatch batch_of(const void* idx, uint32_t index_size, uint64_t n, int has_pad, int64_t pad, float scale, uint64_t stride) {
    RowBatch b;
    b.idx = idx;
    b.index_size = index_size;
    b.has_pad = has_pad != 0;
    b.pad = pad;
    b.n = n;
    b.scale = scale;
    b.stride = stride;
    return b;
}

// the context's device for the launches of one call, the caller's afterwards
struct OnDevice {
    int was = 0;
    bool ok, moved = false;
    explicit OnDevice(int device) {
        ok = hipGetDevice(&was) == hipSuccess;
        if (ok && was != device) ok = moved = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() { if (moved) (void)hipSetDevice(was); }
};
lmr_status_t hip_status(hipError_t e) { return e == hipSuccess ? LMR_OK : LMR_E_HIP; }

}  // namespace
}  // namespace lmr

using namespace lmr;

extern "C" {

lmr_status_t lmr_rows_load(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                           int has_pad, int64_t pad, float scale, void* d_out, uint32_t out_type, uint64_t out_stride,
                           lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_out, out_type, out_stride, false);
    if (st != LMR_OK || n == 0) return st;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_load(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, scale, out_stride), d_out,
                                  out_type, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

uint64_t lmr_rows_add_workspace(const lmr_rows_t* table, uint64_t n) {
    (void)table; (void)n;
    return 0;
}

lmr_status_t lmr_rows_add(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                          int has_pad, int64_t pad, float scale, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                          void* d_work, uint64_t work_bytes, lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_vals, val_type, val_stride, true);
    if (st != LMR_OK) return st;
    if (table->type > LMR_ROW_BF16) return LMR_E_UNSUPPORTED;
    if (n == 0) return LMR_OK;
    if (work_bytes < lmr_rows_add_workspace(table, n) || (work_bytes && (!d_work || !aligned(d_work, 16))))
        return LMR_E_WORKSPACE;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_add(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, scale, val_stride), d_vals,
                                 val_type, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

lmr_status_t lmr_rows_store(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                            int has_pad, int64_t pad, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                            lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_vals, val_type, val_stride, true);
    if (st != LMR_OK || n == 0) return st;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_store(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, 1.f, val_stride), d_vals,
                                   val_type, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
