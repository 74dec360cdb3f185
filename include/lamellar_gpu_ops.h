/*
 * lamellar_gpu_ops.h — C ABI of liblamellar_gpu_ops.so, the MI355X (gfx950)
 * device path for pnnl/lamellar-runtime's LamellarArray batched element ops.
 *
 * Drop-in boundary. The reference's path has two halves,
 * both replaced here, with the op-builder API above them unchanged:
 *
 *   pack  — UnsafeArray::{one_val_multi_indices, multi_val_one_index,
 *           multi_val_multi_index} (src/array/unsafe/operations.rs:479-811)
 *           turn (global index, value) inputs into per-destination-PE op
 *           buffers of IdxVal<I,T> records.          -> lmr_pack
 *   apply — the exec() bodies of the AMs generated by impl/src/array_ops.rs
 *           (:863-1408), looked up through the type-erased registries
 *           MultiValMultiIdxFn / SingleValMultiIdxFn / MultiValSingleIdxFn
 *           (src/array/unsafe/operations.rs:14-18).   -> lmr_apply_{mvmi,svmi,mvsi}
 *   results back to input order — ArrayFetchBatchOpHandle /
 *           ArrayResultBatchOpHandle (src/array/operations/handle.rs:293-325,
 *           495-530).                                  -> lmr_scatter_results
 *   reductions (unsafe.rs:1414-1557, array_reduce.rs)    -> lmr_reduce
 *
 * Beside it, batches whose record is a whole row of a table (no counterpart in the
 * reference): lmr_rows_load / lmr_rows_add / lmr_rows_store.
 *
 * Conventions
 *  - Pointers named d_* are device (HBM) pointers; everything else is host.
 *  - Every device call is stream-ordered and asynchronous; `stream` is a
 *    hipStream_t passed as void* (NULL = the default stream). The library
 *    never allocates or frees on the hot path: workspace is set up by
 *    lmr_ctx_reserve. A context's workspace and pack scratch serve one stream at
 *    a time: calls on one context from different streams must not overlap
 *    (lmr_batch_exchange orders its internal streams itself); use one context
 *    per concurrent stream.
 *  - Errors the reference reports by panicking (out-of-bounds index, integer
 *    division by zero, MIN/-1, op not generated for the element type) are
 *    reported as status codes. Argument errors return immediately; errors
 *    found per element on the device are OR-ed into the context's device
 *    error word (LMR_ERRBIT_*) and read back by lmr_ctx_error. Records that
 *    raise an error are not applied.
 *  - Records within one call are applied atomically per element in an
 *    unspecified order. Fetch results are a valid linearisation (every old
 *    value returned is the element value at some point of a serial order).
 */
#ifndef LAMELLAR_GPU_OPS_H
#define LAMELLAR_GPU_OPS_H

#include "lamellar_types.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LMR_ABI_VERSION 8u

typedef struct lmr_ctx lmr_ctx_t;
typedef void* lmr_stream_t; /* hipStream_t */

/* Apply strategy. AUTO picks ORDERED below 1000 records, DIRECT (one device atomic
 * per record) below 65536 and TILED (LDS-tile apply after counting-sort binning)
 * above. DIRECT and TILED apply every record atomically per element in an
 * unspecified order: one of the outcomes the reference allows for records of
 * different AMs (operations/arithmetic.rs:57-58). ORDERED applies them per element
 * in record order, each element's records as one atomic block: the outcome of the
 * reference's sequential apply loop of one AM (impl/src/array_ops.rs:203-250), so
 * order-dependent ops (swap, store, compare_exchange, rem, floats, fetch results)
 * give exactly the reference's result for a buffer that is one AM. Every 1-PE batch
 * below 1000 records is one AM in the reference (one OpInput chunk,
 * src/array/operations.rs:462-469, less than one AM buffer, unsafe/operations.rs:
 * 679-681); a caller applying one AM's idx_vals of more records (up to 100 kB)
 * asks for ORDERED explicitly. */
typedef enum {
    LMR_STRATEGY_AUTO = 0,
    LMR_STRATEGY_DIRECT = 1,
    LMR_STRATEGY_TILED = 2,
    LMR_STRATEGY_ORDERED = 3
} lmr_strategy_t;

/* What an apply call needs to know about the target array and the op.
 * Mirrors the AM struct fields {data, op} of impl/src/array_ops.rs:852-861:
 * `data` -> (shard, shard_len, kind, dtype), `op: ArrayOpCmd<T>` -> (op,
 * cmp_bits, eps_bits) where CompareExchange(current) / CompareExchangeEps(
 * current, eps) carry their operands as raw little-endian element bits. */
typedef struct {
    void* shard;          /* device pointer: this PE's local slice of the (sub)array */
    uint64_t shard_len;   /* elements in the local slice (num_elems_local) */
    uint32_t kind;        /* lmr_array_kind_t */
    uint32_t dtype;       /* lmr_dtype_t */
    uint32_t op;          /* lmr_opcmd_t (ArrayOpCmd order) */
    uint32_t strategy;    /* lmr_strategy_t */
    uint64_t cmp_bits;    /* CompareExchange(current) */
    uint64_t eps_bits;    /* CompareExchangeEps(_, eps) */
} lmr_apply_desc_t;

/* ---------------------------------------------------------------- misc */
uint32_t lmr_abi_version(void);
const char* lmr_status_string(lmr_status_t status);

/* ---------------------------------------------------------------- context */
/* Per-device context: device error word + pack scratch, and one side stream of its own: a
 * tile sweep forks its hot-tile (delta) kernel onto it and joins it back into the caller's
 * stream before returning (device-scope events; the caller sees one stream). */
lmr_status_t lmr_ctx_create(int device, lmr_ctx_t** out);
lmr_status_t lmr_ctx_destroy(lmr_ctx_t* ctx);
/* Workspace for the tiled apply of up to max_records records per piece;
 * larger batches are processed in pieces. 0 frees the workspace. The old workspace
 * is freed at once: call it when the context's earlier work has completed. A staged session
 * (lmr_stage_*) applies what it holds when the next stream would not fit, so the
 * workspace also sets how many batches one session sweeps together. */
lmr_status_t lmr_ctx_reserve(lmr_ctx_t* ctx, uint64_t max_records);
/* Waits for `stream`, returns the accumulated LMR_ERRBIT_* word in *errbits
 * and the first matching status; clears the word when clear != 0. */
lmr_status_t lmr_ctx_error(lmr_ctx_t* ctx, lmr_stream_t stream, uint32_t* errbits, int clear);

/* Per-kernel timing with HIP events recorded on the caller's stream around
 * every kernel stage this context launches (off by default; events come from
 * a pool created on first use). lmr_ctx_profile_read waits for `stream` and
 * returns accumulated milliseconds, launch counts and records processed per
 * stage (any output may be NULL). */
typedef enum {
    LMR_STAGE_DIRECT = 0,        /* k_apply_direct  */
    LMR_STAGE_MVSI = 1,          /* k_apply_mvsi    */
    LMR_STAGE_BIN_COUNT = 2,     /* k_bin_count     */
    LMR_STAGE_SCAN = 3,          /* scan + tile starts */
    LMR_STAGE_BIN_SCATTER = 4,   /* k_bin_scatter / k_coarse_scatter (+ offsets) */
    LMR_STAGE_TILE_APPLY = 5,    /* plan + k_tile_owner + k_tile_delta */
    LMR_STAGE_PACK = 6,          /* k_pack_count + scan + k_pack_scatter */
    LMR_STAGE_SCATTER_RESULTS = 7,
    LMR_STAGE_FINE_SCATTER = 8,  /* k_fine_scatter  */
    LMR_STAGE_UNPARTITION = 9,   /* k_unpartition: binned results back to input order */
    LMR_STAGE_WINDOW = 10,       /* k_win_count + k_win_scatter: records by shard window (shards above 2^14 tiles) */
    LMR_STAGE_ORDERED = 11,      /* k_order_small / k_order_keys + radix sort + k_order_chains */
    LMR_NUM_STAGES = 12
} lmr_stage_t;
lmr_status_t lmr_ctx_profile(lmr_ctx_t* ctx, int enable);
lmr_status_t lmr_ctx_profile_read(lmr_ctx_t* ctx, lmr_stream_t stream, double* stage_ms,
                                  uint64_t* stage_launches, uint64_t* stage_records, int reset);

/* ---------------------------------------------------------------- host index math
 * src/array/unsafe.rs: async_new :178-274, sub_array :1259-1290,
 * pe_and_offset_for_global_index :1207-1223 (-> :1610-1647, :1651-1736),
 * num_elems_pe :1966-2016, local_as_mut_slice :2023-2066;
 * IndexSize rule src/array/unsafe/operations.rs:56-75, :300-304. */
lmr_status_t lmr_layout_new(lmr_layout_t* L, uint64_t array_size, uint32_t num_pes,
                            uint32_t my_pe, uint32_t distribution);
lmr_status_t lmr_layout_sub(const lmr_layout_t* parent, uint64_t start, uint64_t end,
                            lmr_layout_t* out);
int lmr_pe_and_offset(const lmr_layout_t* L, uint64_t index, uint64_t* pe, uint64_t* offset);
uint64_t lmr_num_elems_pe(const lmr_layout_t* L, uint32_t pe);
uint64_t lmr_local_slice_start(const lmr_layout_t* L, uint32_t pe);
uint32_t lmr_index_size(const lmr_layout_t* L);
/* sizeof(IdxVal<I,T>) and offset of .val (#[repr(C)], src/array/operations.rs:213-219) */
uint32_t lmr_record_bytes(uint32_t index_size, uint32_t dtype);
uint32_t lmr_record_val_offset(uint32_t index_size, uint32_t dtype);
/* BatchReturnType of each op (None / Vals / Result) and op availability per
 * (kind, T) (src/array.rs:207-220, impl/src/array_ops.rs:1503-1533). */
uint32_t lmr_op_ret_kind(uint32_t op);
int lmr_op_supported(uint32_t kind, uint32_t dtype, uint32_t op);

/* ---------------------------------------------------------------- pack
 * Replaces the pack loops of src/array/unsafe/operations.rs:
 * multi_val_multi_index :663-811 (d_vals != NULL) and one_val_multi_indices
 * :479-587 (d_vals == NULL). Global indices (usize) -> (PE, local offset) by
 * the layout, narrowed to index_size bytes. Output: records grouped by
 * destination PE, PE p's records at [d_dest_offsets[p], d_dest_offsets[p+1])
 * in input order (stable), as structure-of-arrays:
 *   d_out_idx  [n] index_size-byte local offsets
 *   d_out_vals [n] values (unused when d_vals == NULL)
 *   d_out_pos  [n] uint32 input positions (the reference's res_buffs), may be NULL
 *   d_dest_counts [num_pes], d_dest_offsets [num_pes + 1]
 * Out-of-bounds indices are dropped and raise LMR_ERRBIT_OOB (the reference
 * panics, :523-526, :716-719). n < 2^32, num_pes <= 512. */
lmr_status_t lmr_pack(lmr_ctx_t* ctx, const lmr_layout_t* layout, const uint64_t* d_gidx,
                      uint64_t n, const void* d_vals, uint32_t dtype, uint32_t index_size,
                      void* d_out_idx, void* d_out_vals, uint32_t* d_out_pos,
                      uint64_t* d_dest_counts, uint64_t* d_dest_offsets, lmr_stream_t stream);
/* Same contract except that records inside one destination's range are in no
 * particular order (d_out_pos still names each record's input position). The
 * device exchange path uses it: the apply does not depend on record order
 * within a buffer (records are applied concurrently, as the reference's AMs
 * are), and the LDS-staged partition behind it writes long per-PE runs. */
lmr_status_t lmr_pack_unordered(lmr_ctx_t* ctx, const lmr_layout_t* layout, const uint64_t* d_gidx,
                                uint64_t n, const void* d_vals, uint32_t dtype, uint32_t index_size,
                                void* d_out_idx, void* d_out_vals, uint32_t* d_out_pos,
                                uint64_t* d_dest_counts, uint64_t* d_dest_offsets, lmr_stream_t stream);

/* Count-free form (the exchange's pack for ops that return nothing): destination p's
 * records go to the fixed region [p * region_cap, (p + 1) * region_cap) of d_out_idx /
 * d_out_vals, unordered, each LDS round reserving its run per destination with one atomic
 * on d_fill[p] (num_pes uint32, zeroed by the call). d_dest_counts[p] = records for PE p;
 * a count above region_cap means that region overflowed and the output is incomplete:
 * pack again with lmr_pack_unordered. num_pes * region_cap < 2^32. */
lmr_status_t lmr_pack_regions(lmr_ctx_t* ctx, const lmr_layout_t* layout, const uint64_t* d_gidx, uint64_t n,
                              const void* d_vals, uint32_t dtype, uint32_t index_size, void* d_out_idx,
                              void* d_out_vals, uint64_t region_cap, uint32_t* d_fill, uint64_t* d_dest_counts,
                              lmr_stream_t stream);

/* ---------------------------------------------------------------- apply
 * d_results: one element per record (for ops whose BatchReturnType is Vals or
 * Result), in record order; d_ok: one byte per record (Result ops: 1 = Ok,
 * 0 = Err). Either may be NULL when the caller does not want them. */

/* MultiValMultiIdxFn (src/array/unsafe/operations.rs:14): d_idx_vals is the
 * reference's op buffer — packed #[repr(C)] IdxVal<I,T> records, I of
 * index_size bytes (impl/src/array_ops.rs:863-899, 1041-1079, 1226-1264); an index_size
 * other than 1, 2 or 4 reads usize (8-byte) records, as the bodies' `_ =>` arm does. */
lmr_status_t lmr_apply_mvmi(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc, const void* d_idx_vals,
                            uint64_t nbytes, uint32_t index_size, void* d_results, uint8_t* d_ok,
                            lmr_stream_t stream);
/* SingleValMultiIdxFn (:15-16): one value (host, element bytes), many local
 * indices of index_size bytes (impl/src/array_ops.rs:929-967, 1109-1149, 1297-1343). */
lmr_status_t lmr_apply_svmi(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc, const void* val,
                            const void* d_indices, uint64_t n, uint32_t index_size,
                            void* d_results, uint8_t* d_ok, lmr_stream_t stream);
/* MultiValSingleIdxFn (:17-18): many values applied in order at one local
 * index, atomically as a block (impl/src/array_ops.rs:235-250, 999-1008). */
lmr_status_t lmr_apply_mvsi(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc, const void* d_vals,
                            uint64_t n, uint64_t index, void* d_results, uint8_t* d_ok,
                            lmr_stream_t stream);
/* Device-native form used after lmr_pack / the RCCL exchange: separate index
 * and value arrays (structure-of-arrays). d_vals == NULL -> the single host
 * value `val` for every record. */
lmr_status_t lmr_apply_soa(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc, const void* d_indices,
                           uint32_t index_size, const void* d_vals, const void* val, uint64_t n,
                           void* d_results, uint8_t* d_ok, lmr_stream_t stream);

/* ---------------------------------------------------------------- staged apply
 * The owner side of the multi-PE exchange. In the reference
 * the op buffers of one batch reach a PE as separate AMs and each is applied on
 * arrival (src/active_messaging/registered_active_message.rs:443-497 ->
 * impl/src/array_ops.rs:863-1408). On the device a batch arrives in chunks (one
 * all-to-all-v each); applying each chunk on arrival would sweep the whole
 * shard once per chunk. A staged session instead partitions every arriving
 * record stream into shard tiles on arrival (lmr_stage_soa) and applies all of
 * them in one sweep of the shard (lmr_stage_finish).
 *   lmr_stage_begin  : open a session for one op on one shard (desc is copied).
 *   lmr_stage_soa    : add n records, lmr_apply_soa's arguments. Their results /
 *                      Ok flags are written to d_results / d_ok (arrival order)
 *                      by the time the session is finished. The records are
 *                      partitioned together with the session's other pending
 *                      streams (one launch per pass for up to 8 streams) at the
 *                      next lmr_stage_flush or lmr_stage_finish: d_indices / d_vals
 *                      must stay valid and unchanged until that call is enqueued.
 *                      Small streams (AUTO, n < 65536) and the DIRECT strategy are
 *                      applied at once; a stream that does not fit the reserved
 *                      workspace first applies what is already staged.
 *   lmr_stage_flush  : partition the pending streams now (their buffers may be
 *                      reused by work enqueued after this call).
 *   lmr_stage_op     : switch the op (and its operands) for later lmr_stage_soa
 *                      calls: a mixed session. Records staged under one op form
 *                      an op phase; phases are applied in staging order per
 *                      element (every record of an earlier phase before any of a
 *                      later one), still in one sweep. A phase of count-free
 *                      regions (order-insensitive ops that return nothing) is
 *                      applied at the switch; later phases are counted regions.
 *                      (On a shard the one-level wide partition covers -- 8-byte
 *                      elements up to 2^24, smaller ones up to 2^26 -- a first
 *                      count-free phase not yet partitioned joins the counted
 *                      phases instead: one partition and one sweep for all.)
 *                      A small stream applied at once first applies the
 *                      phases staged under other ops.
 *   lmr_stage_finish : apply everything staged and close the session.
 * Every call of a session uses one stream; lmr_ctx_reserve is refused while
 * records are staged. Records of one op phase are applied atomically per
 * element in an unspecified order, as within one lmr_apply_soa call. Replaces
 * the reference's per-AM apply of consecutive batches on one array
 * (impl/src/array_ops.rs:863-1408), which gives batches in flight together no
 * order at all; phases in staging order are one of its allowed outcomes. */
lmr_status_t lmr_stage_begin(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc);
lmr_status_t lmr_stage_soa(lmr_ctx_t* ctx, const void* d_indices, uint32_t index_size, const void* d_vals,
                           const void* val, uint64_t n, void* d_results, uint8_t* d_ok, lmr_stream_t stream);
lmr_status_t lmr_stage_op(lmr_ctx_t* ctx, uint32_t op, uint64_t cmp_bits, uint64_t eps_bits, lmr_stream_t stream);
lmr_status_t lmr_stage_flush(lmr_ctx_t* ctx, lmr_stream_t stream);
lmr_status_t lmr_stage_finish(lmr_ctx_t* ctx, lmr_stream_t stream);

/* ---------------------------------------------------------------- exchange (num_pes > 1)
 * The reference moves a batch's op buffers to their owner PEs over a lamellae
 * (trait LamellaeComm / LamellaeAM, src/lamellae.rs:175-221; shmem:
 * Shmem::send_to_pes_async src/lamellae/shmem_lamellae.rs:168-186,
 * CommandQueue::send / recv_data src/lamellae/command_queues.rs:725-807,
 * 1395-1531) and returns fetch results in AM replies
 * (registered_active_message.rs:307-359). Here the transport is a table of two
 * collectives, so a caller can plug its own (as the reference plugs local /
 * shmem / rofi lamellae); lmr_transport_rccl_create builds the MI355X one: RCCL
 * grouped ncclSend / ncclRecv over xGMI on the caller's stream.
 * host_buffers = 1 marks a transport whose callbacks take host memory: the
 * library synchronizes the stream and stages through pinned host buffers around
 * each call (CPU-side collectives, e.g. a gloo process group in tests).
 * flags & LMR_TRANSPORT_SPLIT_HEADERS: `alltoall` (used for the per-chunk header
 * rows only) may run on a stream of its own, concurrently with `alltoallv` on another
 * (the RCCL transport sends headers over a communicator split off its data
 * communicator; host-buffer transports are host-ordered anyway). The exchange then
 * posts chunk j+1's header exchange before chunk j's all-to-all-v, so the host's
 * wait for the counts does not wait for the previous chunk's records. */
#define LMR_TRANSPORT_SPLIT_HEADERS 1u
#define LMR_TRANSPORT_PEER 2u
typedef struct lmr_transport lmr_transport_t;
struct lmr_transport {
    uint32_t num_pes;
    uint32_t my_pe;
    uint32_t host_buffers;
    uint32_t flags;           /* LMR_TRANSPORT_* */
    void* self;
    /* all-to-all: `bytes` at send + p * bytes go to PE p; PE p's arrive at recv + p * bytes */
    lmr_status_t (*alltoall)(void* self, const void* send, void* recv, uint64_t bytes, lmr_stream_t stream);
    /* all-to-all-v: send_bytes[p] bytes at send + send_offs[p] go to PE p; recv_bytes[p]
     * bytes from PE p land at recv + recv_offs[p]; every count and offset is a multiple
     * of `unit` (1, 2, 4 or 8: the element width of the buffer) */
    lmr_status_t (*alltoallv)(void* self, const void* send, const uint64_t* send_bytes, const uint64_t* send_offs,
                              void* recv, const uint64_t* recv_bytes, const uint64_t* recv_offs, uint32_t unit,
                              lmr_stream_t stream);
};

/* RCCL transport: one rank calls lmr_rccl_unique_id and distributes the 128 bytes
 * (the reference's launcher shares its job id the same way, lamellar_run.sh:31-40);
 * every PE then calls lmr_transport_rccl_create (collective, blocking). */
lmr_status_t lmr_rccl_unique_id(uint8_t id[128]);
lmr_status_t lmr_transport_rccl_create(const uint8_t id[128], uint32_t num_pes, uint32_t my_pe, int device,
                                       lmr_transport_t** out);
lmr_status_t lmr_transport_rccl_destroy(lmr_transport_t* tp);
/* The peer-memory transport (collective over the PEs of one node): records pushed straight
 * into the owners' HBM. Every PE allocates receive regions of region_records records
 * (0: one default LAMELLAR_EXCHANGE_CHUNK chunk's region) per source PE and chunk parity
 * (16 B per record) and exports them with hipIpcGetMemHandle; every PE maps every other's.
 * Per-chunk record counts and sequence numbers go through a /dev/shm mailbox named
 * "/lmr_peer_<job>" (job: the same string on every PE, unique per job, no '/') -- the
 * reference's shmem heap (shmem_comm.rs:47-80). lmr_batch_exchange over it pushes: a
 * sender's count-free pack writes each destination's runs into that destination's region,
 * publishes the count, and the owner stages the region once every source has published
 * (device-side waits; one host handshake per batch, no per-chunk host read). Batches the push
 * does not cover (ops that return values, ordered or MVSI batches, regions larger than
 * region_records, the overflow round) use `base`'s collectives, which must stay valid.
 * Pushed chunks of ops the owner stages count-free are packed by (owner PE, owner bucket of 256
 * tiles) into bucket slices of the region, and the owner bins them into its tile regions without
 * a coarse pass (on by default; LAMELLAR_EXCHANGE_BUCKETS=0 on any PE keeps the plain push for
 * the batch: the PEs agree in the handshake). Overflowing records take the overflow round.
 * Receive regions are uncached device memory (LMR_PEER_REGION_MEM=fine: fine-grained instead;
 * plain cached HBM is not offered: a peer's stores do not invalidate the owner's L2), one IPC
 * allocation per (source, parity, index | values) region. Cross-GPU visibility of the pushed
 * stores is unverified until a multi-GPU run checks it; the transport is opt-in.
 * Up to 64 PEs. flags = base->flags | LMR_TRANSPORT_PEER. LAMELLAR_PEER_TIMEOUT (seconds,
 * default 120) bounds every wait: a device wait that times out sets LMR_ERRBIT_TRANSPORT. */
lmr_status_t lmr_transport_peer_create(const lmr_transport_t* base, const char* job, uint64_t region_records,
                                       int device, lmr_transport_t** out);
lmr_status_t lmr_transport_peer_destroy(lmr_transport_t* tp);
/* batches handshaken and chunks pushed so far (either output may be NULL) */
lmr_status_t lmr_transport_peer_stats(const lmr_transport_t* tp, uint64_t* batches, uint64_t* pushed_chunks);

/* One batched op over all PEs, collective: every PE calls it with its own batch (a PE
 * with nothing to send passes i_len = 0). Replaces, for num_pes > 1,
 * UnsafeArray::initiate_batch_op / _fetch_op_2 / _result_op_2
 * (src/array/unsafe/operations.rs:290-477) with the AMs' trip over the lamellae:
 *   pack by owner PE -> per-PE header all-to-all (count, MVSI local index, flags, scalar
 *   value, chunk count) -> all-to-all-v of local indices and values -> the owner stages
 *   every arriving stream (lmr_stage_*) and applies all in one shard sweep -> reverse
 *   all-to-all-v of results -> lmr_scatter_results into input order
 *   (operations/handle.rs:315-317).
 * Order. A batch of fewer than 1000 records (AUTO), or any batch with
 * desc->strategy == LMR_STRATEGY_ORDERED, is one reference AM per destination: its
 * records reach each owner in input order (stable pack) and the owner applies them in
 * that order, each element's records of one stream as one atomic block -- the outcome of
 * the reference's sequential apply of each source's AM (unsafe/operations.rs:709-758,
 * impl/src/array_ops.rs:203-250). Streams of different sources are applied one after
 * another in PE order (the reference applies concurrent AMs in no fixed order; one source
 * order is one of its outcomes). Larger AUTO batches are applied atomically per element
 * in an unspecified order (a linearisation), as the reference's concurrently applied AMs.
 * The batch is cut into chunks of LAMELLAR_EXCHANGE_CHUNK records (default 2^26, at
 * most 2^27), pipelined over three internal streams (pack; forward collectives; owner
 * apply and the reverse collectives). A failed transport call ends the exchange with
 * its status; an RCCL transport is aborted first (ncclCommAbort: its queued peer calls
 * can never complete) and refuses every later call, so the job must build a new one;
 * everything is ordered after and before `stream`. Index forms as the op builders:
 * i_len == 1 takes the global index h_index (host); otherwise d_gidx holds i_len
 * global indices (usize). Values: v_len == 1 takes the host element h_val (SVMI /
 * single), otherwise d_vals holds v_len elements; i_len == 1 with v_len > 1 is MVSI
 * (applied at the owner as one atomic block). desc->shard / shard_len: this PE's
 * local slice; the workspace (lmr_ctx_reserve) should hold the records this PE
 * receives (more are applied in several sweeps). The host reads chunk 0's header rows
 * (RCCL's all-to-all-v takes host counts). Fixed-region mode (ops that return nothing,
 * every PE packing count-free and staging count-free, LAMELLAR_EXCHANGE_FIXED unset or 1):
 * each destination's fixed region goes whole, the owner stages it with its record count
 * read on the device from the header rows, and the host reads no later chunk's rows;
 * records that did not fit their region are exchanged once more after the last chunk.
 * Otherwise the host reads every chunk's rows while the next chunk is packed. */
lmr_status_t lmr_batch_exchange(lmr_ctx_t* ctx, const lmr_transport_t* tp, const lmr_layout_t* layout,
                                const lmr_apply_desc_t* desc, const uint64_t* d_gidx, uint64_t h_index,
                                uint64_t i_len, const void* d_vals, const void* h_val, uint64_t v_len,
                                void* d_results, uint8_t* d_ok, lmr_stream_t stream);

/* Deferred exchange sessions. With lmr_ctx_exchange_defer(ctx, 1), an lmr_batch_exchange of an
 * op that returns nothing, whose owner-side session is count-free, leaves that session open: the
 * records this PE received are partitioned into the workspace (the callers' and the transport's
 * buffers are free when the call completes) but the shard sweep has not run. The next
 * lmr_batch_exchange with the same descriptor adds its records to the open session (the session
 * sweeps whenever the workspace fills), and lmr_exchange_flush applies what is staged, in
 * `stream` order: one sweep for several batches, as the deferred 1-PE sessions do (the
 * reference's batches are asynchronous until wait_all, src/array/operations.rs). Any other
 * lmr_batch_exchange applies the open session first. The shard must not be read, written or freed
 * before lmr_exchange_flush (a new shard at the same address would continue the session); a
 * failed exchange drops the open session's records. While a deferred session is open the
 * context's workspace holds its records, so every other use of the workspace applies it first, in
 * the call's stream order (lmr_apply_soa / _svmi / _mvmi / _mvmi_host, lmr_apply_msg), and the
 * staged-session calls (lmr_stage_begin / _soa / _op / _flush / _finish) return LMR_E_INVALID until
 * lmr_exchange_flush has run.
 * lmr_exchange_flush with no deferred session open does nothing. Deferral is off by default. */
lmr_status_t lmr_ctx_exchange_defer(lmr_ctx_t* ctx, int on);
lmr_status_t lmr_exchange_flush(lmr_ctx_t* ctx, lmr_stream_t stream);

/* The exchange's host planning of one chunk, exported for tests (pure host code).
 * Header rows are LMR_XHDR_WORDS int64 per PE: [count, MVSI local index or -1, flags
 * (LMR_XHDR_SCALAR: one scalar value; LMR_XHDR_ORDERED: an in-order stream; LMR_XHDR_FIXED:
 * the sender packs fixed per-destination regions; LMR_XHDR_OVERFLOW: the sender's overflow list
 * is not empty so far (its last chunk's rows decide whether the batch needs the overflow round);
 * LMR_XHDR_DEVCOUNT: the PE stages fixed
 * regions with device-side counts; LMR_XHDR_BUCKETS: the sender's fixed regions are laid out by
 * owner bucket -- a header of slice counts, then the slices -- and go whole), the scalar's bits, the sender's chunk count, the
 * sender's packed records in the batch, its chunk size in records]. From the rows this
 * PE sent (send_hdr, row p to PE p) and received (recv_hdr, row p from PE p): byte
 * splits / offsets of the index (iw-byte) and value (eb-byte) all-to-all-v's -- MVSI
 * senders send no index, scalar senders no values -- into caller arrays of num_pes
 * entries. Returns the batch's chunk count (the largest any PE announced). */
#define LMR_XHDR_WORDS 7
#define LMR_XHDR_SCALAR 1
#define LMR_XHDR_ORDERED 2
#define LMR_XHDR_FIXED 4
#define LMR_XHDR_DEVCOUNT 8
#define LMR_XHDR_OVERFLOW 16
#define LMR_XHDR_BUCKETS 32
uint64_t lmr_exchange_plan(uint32_t num_pes, uint32_t iw, uint32_t eb, const int64_t* send_hdr,
                           const int64_t* recv_hdr, uint64_t* idx_sb, uint64_t* idx_so, uint64_t* idx_rb,
                           uint64_t* idx_ro, uint64_t* val_sb, uint64_t* val_so, uint64_t* val_rb,
                           uint64_t* val_ro);

/* ---------------------------------------------------------------- host buffers
 * Host-buffer ingestion: the op buffer is the
 * reference's own IdxVal<I,T> bytes in host memory (the AM body in the shmem
 * lamellae heap, src/lamellae/shmem/shmem_comm.rs:302-352; deserialised in
 * src/active_messaging/registered_active_message.rs:443-497), and fetch
 * results / Ok flags land in host memory (the AM's returned Vec<T>).
 * lmr_host_register records a host range as an op / result buffer; caller memory is never
 * page-locked by the library (every pattern of locking, unlocking and freeing it that earlier
 * rounds tried was followed, on some runs, by a device fault at a later copy), so copies of a
 * registered range are staged through the bounce slots like any pageable buffer. A range
 * overlapping an earlier range's bytes, or lmr_host_unregister with a pointer that does not
 * start a registration, is refused with LMR_E_INVALID. lmr_host_registered reports a
 * registered range as (0, 0, 1): no pinned pages. For zero-copy DMA the buffers come from
 * lmr_host_alloc (the reference's lamellae heap, mapped once at world init and dropped at
 * shutdown, shmem_comm.rs:47-80); lmr_host_alloc / lmr_host_free
 * give short-lived pinned buffers (hipHostMalloc; free waits for the library's host
 * copies); they, and any memory the runtime allocated pinned, are DMA'd in place
 * without registration. lmr_apply_mvmi_host uploads
 * the records in pieces (LMR_HOST_PIECE_RECORDS, default 2^22), applies each piece on
 * `stream` while the next uploads and the previous one's results download, and
 * orders completion of everything (results included) on `stream`. Buffers the runtime
 * did not allocate pinned (pageable or registered caller memory) go through the library's
 * pinned bounce slots: records are copied on the host before their upload, and results /
 * Ok flags bound for them are written by the host before the call returns. The host
 * buffers must stay untouched until `stream` completes. Records up to 16 bytes. */
lmr_status_t lmr_host_register(void* ptr, uint64_t bytes);
lmr_status_t lmr_host_unregister(void* ptr);
/* A lamellae heap ("hipHostRegister of the shmem heap"): the whole pages inside
 * [ptr, ptr + bytes) are page-locked once, for the heap's lifetime (the reference maps its heap
 * at world init and drops it at shutdown, shmem_comm.rs:47-80); copies of buffers inside it DMA
 * those pages in place and stage the partial end pages. lmr_host_unregister_heap unlocks it
 * (after the library's in-flight host copies): call it at shutdown only -- unlocking and freeing
 * host memory while the process goes on copying is the pattern that preceded every host-path
 * fault on this pool. lmr_host_registered reports a heap's pinned pages. */
lmr_status_t lmr_host_register_heap(void* ptr, uint64_t bytes);
lmr_status_t lmr_host_unregister_heap(void* ptr);
lmr_status_t lmr_host_registered(const void* ptr, uint64_t bytes, uint64_t* pin_base, uint64_t* pin_bytes,
                                 uint32_t* ranges);
lmr_status_t lmr_host_alloc(uint64_t bytes, void** out);
lmr_status_t lmr_host_free(void* ptr);
lmr_status_t lmr_apply_mvmi_host(lmr_ctx_t* ctx, const lmr_apply_desc_t* desc, const void* h_idx_vals,
                                 uint64_t nbytes, uint32_t index_size, void* h_results, uint8_t* h_ok,
                                 lmr_stream_t stream);

/* ---------------------------------------------------------------- results
 * d_out[d_pos[k]] = d_in[k] (and d_ok_out[d_pos[k]] = d_ok_in[k] when both are
 * non-NULL): handle.rs:315-317 `results[res_buff[k]] = res[k]`. */
lmr_status_t lmr_scatter_results(const void* d_in, const uint32_t* d_pos, uint64_t n,
                                 uint32_t elem_bytes, void* d_out, const uint8_t* d_ok_in,
                                 uint8_t* d_ok_out, lmr_stream_t stream);

/* ---------------------------------------------------------------- reduce
 * The per-PE step of UnsafeArray::reduce / sum / prod / max / min
 * (src/array/unsafe.rs:1414-1557): the reduction AM's
 * `local_data().iter().reduce(op)` (impl/src/array_reduce.rs:82-88) over the
 * len elements at d_shard. d_out receives the result's bits (8 bytes, element in
 * the low bytes); *d_has = 0 for an empty slice (the reference's None). The
 * cross-PE tree (:90-107) combines the PEs' (has, value) pairs. Integer ops
 * wrap; float sum / prod are folded in a tree order (rounding may differ from
 * the sequential fold); max / min are exact (NaN order unspecified). */
lmr_status_t lmr_reduce(lmr_ctx_t* ctx, uint32_t dtype, uint32_t op, const void* d_shard, uint64_t len,
                        uint64_t* d_out, uint8_t* d_has, lmr_stream_t stream);

/* ---------------------------------------------------------------- rows
 * The batched load / add / store with a whole row as the record: a table of `rows` rows of
 * row_len elements in HBM, a batch of n row indices and (add, store) n rows of values. This PE's
 * rows only; a table over several PEs packs its records by owner first (lmr_pack) and calls these
 * at the owner.
 *   d_idx       n row indices, signed, 4 or 8 bytes each (index_size). An index equal to `pad`
 *               (has_pad != 0) names no row: load writes zeros, add and store skip the record.
 *               Any other index outside [0, rows) does the same and raises LMR_ERRBIT_OOB.
 *   values      n rows of row_len elements of val_type / out_type (LMR_ROW_F32, _F16 or _BF16),
 *               `stride` elements apart; add and store also take stride 0: one row for every record.
 *               They must not overlap the table.
 * Arithmetic is f32, rounded once (to nearest, ties to even) where a narrower type is written.
 * Nothing is allocated and nothing waits; every call may be captured into a graph. They use none of
 * the context's workspace (only its device and error word; no stage timing): calls on different tables may run on
 * several streams at once, calls that write one table must be ordered by the caller. n <= LMR_ROW_MAX_BATCH, n * row_len <= LMR_ROW_MAX_VALUES,
 * stride <= LMR_ROW_MAX_STRIDE. */
#define LMR_ROW_MAX_LEN (1u << 18)
#define LMR_ROWS_MAX 0xFFFFFFF0ull
#define LMR_ROW_MAX_BATCH (1ull << 25)
#define LMR_ROW_MAX_VALUES (1ull << 36)
#define LMR_ROW_MAX_STRIDE 0xFFFFFFFFull
#define LMR_ROW_SCAN 1024u
typedef struct {
    void* data;          /* device pointer: row r starts at element r * row_len */
    float* scales;       /* 8-bit types: rows x (row_len / group) scales; otherwise unused */
    uint32_t* claims;    /* rows words, zero before the first lmr_rows_store that uses them and left
                            zero by each; used by stores of more than LMR_ROW_SCAN records, where
                            NULL says that no row occurs twice */
    uint64_t rows;       /* <= LMR_ROWS_MAX */
    uint64_t row_len;    /* 1 .. LMR_ROW_MAX_LEN elements */
    uint32_t type;       /* lmr_row_type_t */
    uint32_t group;      /* 8-bit types: elements per scale, divides row_len */
} lmr_rows_t;
/* out[t, :] = scale * table[idx[t], :] (8-bit tables: scale * (code * its group's scale)) */
lmr_status_t lmr_rows_load(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                           int has_pad, int64_t pad, float scale, void* d_out, uint32_t out_type, uint64_t out_stride,
                           lmr_stream_t stream);
/* table[r, :] += scale * (sum of vals[t, :] over the records t of row r), for every row named: the
 * records of a row are summed in f32 in an order that the indices alone decide, so equal calls give
 * equal bits. Tables of 8-bit codes: LMR_E_UNSUPPORTED. d_work: lmr_rows_add_workspace bytes
 * (16-byte aligned), the call's own until it has run on the stream; LMR_E_WORKSPACE when short. */
uint64_t lmr_rows_add_workspace(const lmr_rows_t* table, uint64_t n);
lmr_status_t lmr_rows_add(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                          int has_pad, int64_t pad, float scale, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                          void* d_work, uint64_t work_bytes, lmr_stream_t stream);
/* table[idx[t], :] = vals[t, :]; of several records of one row the last one is stored. 8-bit
 * tables: per group, scale = max(max|x| / Q, 2^-126) with Q = 127 (I8) or 448 (E4M3) and code =
 * x / scale rounded to the nearest code, each rounding in f32; an infinity or NaN makes the group's
 * scale NaN. */
lmr_status_t lmr_rows_store(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                            int has_pad, int64_t pad, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                            lmr_stream_t stream);

/* ---------------------------------------------------------------- AM wire format
 * The op AMs as the running runtime puts them in a lamellae buffer (SURVEY.md 8(a)
 * a17, 8(f) ranks 1 and 4): bincode legacy (little endian, fixed-width integers,
 * usize = u64, enum tags u32, Option tag u8, byte vectors u64 length + bytes;
 * src/lib.rs:319-321). A message is Option<SerializeHeader{Msg{src: u16, cmd: Cmd}}>
 * (src/lamellae.rs:102-104, 33-34) followed by its data:
 *   Cmd::Am        : AmHeader{am_id: i32, team_addr: usize, req_id: ReqId{id, sub_id}}
 *                    (registered_active_message.rs:80-85, 278-300) + the AM struct;
 *   Cmd::BatchedMsg: entries [Cmd][header][body] back to back (simple_batcher.rs:327-489),
 *                    Cmd::Am / ReturnAm entries as above, Cmd::Data = DataHeader{size,
 *                    req_id, darc_list_size} + darc list + data, Cmd::Unit = UnitHeader{req_id}.
 * The op AM structs (impl/src/array_ops.rs:855-861, 920-927, 991-997 and their _fetch /
 * _result twins) are {data: the array handle, op: ArrayOpCmd<T>, then MVMI idx_vals:
 * bytes, index_size: u8 | SVMI val: T, indices: bytes, index_size: u8 | MVSI vals: bytes,
 * index: usize}. The array handle by kind: UnsafeArray / ReadOnlyArray = UnsafeArrayInner
 * {data: Darc, distribution, orig_elem_per_pe, orig_remaining_elems, elem_size, offset,
 * size, sub: bool} (unsafe.rs:106-116); NativeAtomicArray = that + orig_t:
 * NativeAtomicType (native_atomic.rs:819-822); GenericAtomicArray / LocalLockArray /
 * GlobalLockArray = a lock Darc first (generic_atomic.rs:272-275, local_lock_atomic.rs:50-53,
 * global_lock_atomic.rs:43-46). Every Darc travels as __NetworkDarc{inner_addr: usize,
 * backend: Backend, orig_world_pe: usize, orig_team_pe: usize} (darc.rs:227-234,
 * 1838-1843). No reference test pins these bytes: the layout is restated from the serde
 * derives, not checked against bytes the reference produced. */
/* LMR_SHAPE_FOREIGN marks a message entry that is not an op AM (a ReturnAm or any other
 * AM): the parse steps over it, lmr_apply_msg leaves it to the runtime. */
typedef enum { LMR_SHAPE_MVMI = 0, LMR_SHAPE_SVMI = 1, LMR_SHAPE_MVSI = 2, LMR_SHAPE_FOREIGN = 3 } lmr_am_shape_t;
typedef enum {   /* Cmd, src/active_messaging.rs:893-902 */
    LMR_CMD_AM = 0, LMR_CMD_RETURN_AM = 1, LMR_CMD_DATA = 2, LMR_CMD_UNIT = 3, LMR_CMD_BATCHED = 4
} lmr_cmd_t;

typedef struct {
    uint64_t inner_addr;
    uint32_t backend;          /* Backend tag as compiled (Local / Shmem [/ Rofi]) */
    uint32_t reserved_;
    uint64_t orig_world_pe;
    uint64_t orig_team_pe;
} lmr_net_darc_t;

typedef struct {
    uint32_t shape, kind, dtype, op;    /* op: the ArrayOpCmd tag (= lmr_opcmd_t) */
    uint64_t cmp_bits, eps_bits;        /* CompareExchange(current) / CompareExchangeEps(current, eps) */
    lmr_net_darc_t data;                /* the array's data Darc */
    lmr_net_darc_t lock;                /* Generic locks / LocalLock / GlobalLock Darc, else zero */
    uint32_t native_type;               /* NativeAtomicType tag (NativeAtomicArray), else 0xFFFFFFFF */
    uint32_t distribution;
    uint64_t orig_elem_per_pe, orig_remaining_elems, elem_size, offset, size;
    uint32_t sub;
    uint32_t index_size;                /* MVMI / SVMI */
    uint64_t val_bits;                  /* SVMI: the value */
    uint64_t index;                     /* MVSI: the local index */
    uint64_t recs_offset, recs_bytes;   /* idx_vals / indices / vals inside the decoded buffer */
    uint64_t body_bytes;                /* serialized size of the AM struct */
} lmr_am_view_t;

/* Decode one op AM struct of (shape, array kind, dtype) from body[0..len). */
lmr_status_t lmr_am_decode(const uint8_t* body, uint64_t len, uint32_t shape, uint32_t kind, uint32_t dtype,
                           lmr_am_view_t* out);
/* Encode one (the sender's side; recs = the records, v->recs_bytes long). *written = bytes
 * (also when out is NULL or cap too small: then LMR_E_LENGTH). */
lmr_status_t lmr_am_encode(const lmr_am_view_t* v, const void* recs, uint8_t* out, uint64_t cap,
                           uint64_t* written);

/* One entry of a message: an AM (body at msg + body_offset), a Data or Unit reply. */
typedef struct {
    uint32_t cmd;
    uint32_t src;
    int32_t am_id;
    uint32_t shape, kind, dtype;        /* from the resolver (AM entries) */
    uint64_t team_addr, req_id, req_sub_id;
    uint64_t body_offset, body_bytes;   /* AM struct / Data bytes (after their header) */
} lmr_msg_entry_t;
/* Called for every Cmd::Am / Cmd::ReturnAm entry with its AmHeader's am_id and the bytes
 * after the header (body[0..avail)). Returns
 *   0: a registered op AM of (shape, kind, dtype) -- the library decodes and sizes it;
 *   1: another AM (a ReturnAm, a user AM): *body_bytes = its serialized size, as the
 *      runtime's own deserializer for am_id finds it (AMS_EXECS, registered_active_message.rs
 *      :443-497); the entry is reported with shape LMR_SHAPE_FOREIGN and stepped over;
 *   anything else: unknown -- the parse stops with LMR_E_UNSUPPORTED.
 * So a batched message mixing op AMs with user AMs, ReturnAms, Data and Unit entries, as the
 * reference's SimpleBatcher builds them (simple_batcher.rs:276-304), parses whole. */
typedef int (*lmr_am_resolver_t)(void* user, uint32_t cmd, int32_t am_id, const uint8_t* body, uint64_t avail,
                                 uint32_t* shape, uint32_t* kind, uint32_t* dtype, uint64_t* body_bytes);
/* msg[0..len) starts at the Option<SerializeHeader> (ShmemData::header_and_data_as_bytes,
 * shmem_comm.rs:640-690). *n = entries (LMR_E_LENGTH when more than cap). */
lmr_status_t lmr_msg_parse(const uint8_t* msg, uint64_t len, lmr_am_resolver_t resolve, void* user,
                           lmr_msg_entry_t* entries, uint32_t cap, uint32_t* n);

/* The reply body of a returning op AM (what its exec returns, bincode): Vec<T> = u64 len +
 * elements (fetch), Vec<Result<T,T>> = u64 len + per element (u32 tag Ok 0 / Err 1, T). */
uint64_t lmr_reply_bytes(uint32_t dtype, uint32_t ret_kind, uint64_t n);
lmr_status_t lmr_reply_encode(uint32_t dtype, uint32_t ret_kind, uint64_t n, const void* results, const uint8_t* oks,
                              uint8_t* out, uint64_t cap);

/* The owner side of a message from the running runtime:
 * every op AM of a single or batched message applied on the device. Small AMs are
 * aggregated: the AMs of one message that name the same shard, op, operands, index width
 * and (SVMI) value are applied as ONE record stream (one upload, one apply) instead of one
 * launch each -- the device counterpart of the reference's small-AM batcher
 * (simple_batcher.rs:65-117, exec_batched_msg :276-304). MVSI AMs keep their block
 * semantics (each applied as one atomic block). shards(v) names the device shard of each
 * decoded AM (NULL shard: skipped); LMR_SHAPE_FOREIGN entries, Data and Unit entries are
 * left to the runtime. Returning AMs get their reply body (lmr_reply_encode)
 * at replies + reply_offs[e], reply_lens[e] bytes, for entry e (reply_offs[e] = ~0 and
 * reply_lens[e] = 0 for entries without one); replies must hold the sum of their
 * lmr_reply_bytes. Synchronous: returns when the
 * replies are written. Order between AMs is unspecified, as for concurrently executing
 * AMs in the reference. */
typedef struct {
    void* shard;
    uint64_t shard_len;
    uint32_t strategy;
    uint32_t reserved_;
} lmr_shard_t;
typedef int (*lmr_shard_resolver_t)(void* user, const lmr_am_view_t* v, lmr_shard_t* out);
lmr_status_t lmr_apply_msg(lmr_ctx_t* ctx, const uint8_t* msg, uint64_t len, lmr_am_resolver_t resolve,
                           lmr_shard_resolver_t shards, void* user, uint8_t* replies, uint64_t reply_cap,
                           uint64_t* reply_offs, uint64_t* reply_lens, uint32_t max_entries, uint32_t* n_entries,
                           lmr_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* LAMELLAR_GPU_OPS_H */
