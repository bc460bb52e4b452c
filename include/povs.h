/*
 * C ABI of the B200-native POV shuffle (libpovs_sm100.so).
 *
 * Every entry point takes plain pointers and sizes, returns 0 on success or a
 * negative POVS_ERR_* code, never terminates the process, and records a
 * message retrievable with povs_last_error_string() (per calling thread).
 * Device work is enqueued on the caller's stream (a cudaStream_t passed as
 * void*; NULL means the legacy default stream) and is asynchronous unless
 * stated otherwise.  The caller owns every data buffer; the library only keeps
 * a small per-device context (a status word and cached CUDA graphs), created
 * on first use and freed by povs_release_v1().
 *
 * Rows ("instances") are opaque byte vectors of row_bytes bytes; the deck is
 * n_rows rows, contiguous.  Shuffling is in place along axis 0.
 */
#ifndef POVS_H
#define POVS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
#define POVS_OK 0
#define POVS_ERR_INVALID_ARGUMENT (-1) /* a size, option or pointer is out of range */
#define POVS_ERR_UNSUPPORTED (-2)      /* valid for the algorithm but outside this library's limits */
#define POVS_ERR_CUDA (-3)             /* a CUDA runtime call failed */
#define POVS_ERR_DEVICE_STATUS (-4)    /* a kernel reported a failure through the device status word */

/* Device status bits reported by povs_device_status_v1(). */
#define POVS_DEV_WAIT_TIMEOUT 1 /* an async-copy barrier wait gave up after its time limit */
#define POVS_DEV_BAD_INJECTED 2 /* an injected permutation entry was out of range and was ignored */

/* Flags of povs_shuffle_v1(). */
/* Launch the iterations one by one (by default decks under 32 MiB replay a cached CUDA graph and
 * larger decks are launched one by one). */
#define POVS_FLAG_NO_GRAPH 1u
#define POVS_FLAG_SYNC 2u     /* synchronize the stream and check the device status before returning */
/* Draw the randomness with the distribution of the reference's CUDA path (per-vblock seeds 1..999,
 * xorshift32 forward Fisher-Yates, padding in the last vblock; src/povs/__cuda/lib/povs.cu:396-430,
 * 294-316) instead of uniform per-vblock permutations.  For statistical comparisons with it. */
#define POVS_FLAG_REFERENCE_RNG 4u
/* Order the iteration kernels with ordinary stream order instead of programmatic dependent
 * launches (by default each iteration kernel's CTAs start their set-up while the kernel before it
 * on the stream drains - the previous iteration, or for decks of 32 MiB and more the previous
 * call's last iteration - and wait for it to complete before touching the deck). */
#define POVS_FLAG_NO_PDL 8u
/* Draw the randomness with the distribution of the reference's NumPy path (padding ids anywhere,
 * members in slot order, per-vblock seeds 1..999 and numpy.random.RandomState(seed).shuffle of the
 * vblock's rows; src/povs/numpy.py:43-61,125-136).  The permutations come from tables built on the
 * host once per (P, V, n_rows % P) and device (at most 128 MiB; a larger geometry is rejected with
 * POVS_ERR_UNSUPPORTED), freed by povs_release_v1.  Excludes POVS_FLAG_REFERENCE_RNG. */
#define POVS_FLAG_REFERENCE_NUMPY 16u

/* Limits of this library. */
#define POVS_MAX_OFFSETS 256 /* offsets are passed to the device inline in the launch parameters */
#define POVS_MAX_VBLOCK 32   /* one warp lane per member pblock */
#define POVS_MAX_VP 1024     /* V * P rows per vblock: one warp sorts the permutation in registers */

/*
 * Shuffle a deck in place: `iterations` POV iterations, all randomness drawn on
 * the device from `seed` (Philox4x32-10 counters: offset choice, a keyed
 * bijection of pblocks onto vblock slots, per-vblock permutations).
 *
 * Replaces the reference's native entry `torch_binding(X, O, iterations,
 * pblock, vblock, block_size, seed)` (src/povs/_cuda.pyi:9-17,
 * src/povs/__cuda/binds/torch.cpp:19-60) and the host loop it dispatches to
 * (src/povs/__cuda/lib/povs.cu:356-467).  Differences: the device pointer and
 * the row size replace the typed tensor (any dtype); offsets are a host array;
 * the GPU thread-block size is not needed; the stream is explicit; errors are
 * return codes instead of exit().
 *
 *   data        device pointer to n_rows * row_bytes bytes
 *   offsets     host array of n_offsets (1..POVS_MAX_OFFSETS) row offsets, each in [0, n_rows)
 *   pblock      P, a power of two >= 1;  vblock: V, a power of two in [2, POVS_MAX_VBLOCK]
 *   device      CUDA ordinal the data lives on
 *   stream      cudaStream_t of that device, or NULL
 */
int povs_shuffle_v1(void* data, int64_t n_rows, int64_t row_bytes, const int64_t* offsets, int32_t n_offsets,
                    int32_t iterations, int32_t pblock, int32_t vblock, uint64_t seed, int32_t device, void* stream,
                    uint32_t flags);

/*
 * Same as povs_shuffle_v1 for a deck in HOST memory: the rows are copied to a
 * device buffer supplied by the caller (`device_buffer`, at least n_rows *
 * row_bytes bytes on `device`), shuffled there and copied back, all on
 * `stream`, and the call returns after the stream has synchronized.  Pinned
 * host memory gives full PCIe / C2C bandwidth; pageable memory works.
 *
 * Serves the reference's CPU route (`povs.shuffle` on a numpy array or a CPU
 * tensor, src/povs/__init__.py:36-42 -> src/povs/numpy.py:18-61) on the GPU.
 */
int povs_shuffle_host_v1(void* host_data, void* device_buffer, int64_t n_rows, int64_t row_bytes,
                         const int64_t* offsets, int32_t n_offsets, int32_t iterations, int32_t pblock,
                         int32_t vblock, uint64_t seed, int32_t device, void* stream, uint32_t flags);

/*
 * Same as povs_shuffle_v1 for a deck that STAYS in host memory, for decks larger than the
 * device's memory: the kernels read and write the rows in place over PCIe / C2C through mapped
 * page-locked memory (plain vector loads and stores, no TMA).  Memory from cudaHostAlloc /
 * cudaMallocHost or already registered is used as is; any other host range is page-locked and
 * mapped for the duration of the call (cudaHostRegister of the enclosing pages) and released
 * before returning.  The call returns after the stream has synchronized.  Throughput is bound by
 * the interconnect (each iteration moves the deck across it twice).
 * Serves the reference's roadmap item of decks larger than memory (CONTRIBUTING.md:16) on the
 * reference's CPU route (src/povs/numpy.py:18-61).
 */
int povs_shuffle_mapped_v1(void* host_data, int64_t n_rows, int64_t row_bytes, const int64_t* offsets,
                           int32_t n_offsets, int32_t iterations, int32_t pblock, int32_t vblock, uint64_t seed,
                           int32_t device, void* stream, uint32_t flags);

/*
 * Shuffle n_decks host decks of the same shape through n_buffers device buffers (>= 2 for
 * overlap; each at least n_rows * row_bytes bytes on `device`): deck d is copied into buffer
 * d % n_buffers, shuffled with seeds[d], and copied back, on internal streams ordered by events so
 * that deck d's copy back overlaps deck d+1's copy in and iterations (the PCIe directions and the
 * SMs work at the same time).  Work queued on `stream` before the call is ordered first; the call
 * returns when every deck is back in host memory.  A host deck may appear more than once in the
 * list (it is then shuffled again, after its previous copy back).  Use pinned host memory for
 * overlap.  Batched form of povs_shuffle_host_v1 (same reference route).
 */
int povs_shuffle_host_batch_v1(void* const* host_decks, int32_t n_decks, void* const* device_buffers, int32_t n_buffers,
                               int64_t n_rows, int64_t row_bytes, const int64_t* offsets, int32_t n_offsets,
                               int32_t iterations, int32_t pblock, int32_t vblock, const uint64_t* seeds,
                               int32_t device, void* stream, uint32_t flags);

/*
 * Apply externally supplied randomness (test hook for bit-exact parity with the
 * reference's CPU and CUDA paths).  For each iteration t:
 *   offsets_per_iter[t]        (host)   the iteration's row offset, in [0, n_rows)
 *   assign + t*n_v*V           (device) int64 [n_v][V] member pblock ids; values < 0 or
 *                                       >= ceil(n_rows/P) are padding
 *   perms  + t*n_v*V*P         (device) int32 [n_v][V*P]; destination slot f of a vblock
 *                                       receives source slot perms[f] (f < valid rows)
 * sort_members = 1 orders each vblock's members ascending with padding last, as the
 * reference kernel does (src/povs/__cuda/lib/povs.cu:203-221); 0 keeps the given order
 * (the NumPy path, src/povs/numpy.py:120-136), except that padding goes last and a
 * truncated last pblock is placed after the full ones.
 * n_v = ceil(ceil(n_rows/P)/V).  Replaces no single reference function: it is the
 * reference kernel's body (povs.cu:116-349) with the host RNG (povs.cu:415-431) cut out.
 */
int povs_apply_v1(void* data, int64_t n_rows, int64_t row_bytes, int32_t pblock, int32_t vblock,
                  int32_t iterations, const int64_t* offsets_per_iter, const int64_t* assign, const int32_t* perms,
                  int32_t sort_members, int32_t device, void* stream);

/*
 * Shuffle a deck stored as up to POVS_MAX_SHARDS shards (one process, one device): rows
 * [sum(shard_rows[0..i-1]), +shard_rows[i]) live at shard_ptrs[i].  The result equals
 * povs_shuffle_v1 on the concatenated deck with the same seed.  Every shard must be addressable
 * from `device` (allocations on it, or peer memory with peer access enabled) and hold at least
 * `pblock` rows; the caller orders any writes to the shards before the call.  scratch_ptrs is NULL
 * (in place: each vblock is read into shared memory and written back) or one buffer per shard of
 * the same size (double-buffered "push" order: each pblock's rows are read once from the buffer
 * holding them and stored straight into their destination slots in the other buffer; an odd
 * number of iterations ends with a copy back).  Both orders give the same result.
 * No reference counterpart: the reference shuffles one contiguous tensor (src/povs/torch.py:20-50).
 */
int povs_shuffle_shards_v1(void* const* shard_ptrs, void* const* scratch_ptrs, const int64_t* shard_rows,
                           int32_t n_shards, int64_t row_bytes, const int64_t* offsets, int32_t n_offsets,
                           int32_t iterations, int32_t pblock, int32_t vblock, uint64_t seed, int32_t device,
                           void* stream, uint32_t flags);

/*
 * Sharded mode, one process per GPU, over the deck whose shards are shard_ptrs (this rank's own
 * shard and the peers' shards as mapped into this process with povs_ipc_import_v1).  With
 * scratch_ptrs NULL, rank `rank` reads the vblocks rank, rank + n_shards, ... from local or peer
 * memory (bulk copies over NVLink, no multicast) and writes them back with peer stores.  With one
 * scratch buffer per shard (same sizes, mapped the same way), rank `rank` moves the pblocks stored
 * in its own shard, reading them locally and storing every row straight into its destination slot
 * in the other buffer, so a row crosses NVLink at most once per iteration (half the traffic).
 * A device barrier over the ranks' flag arrays (peer_flags[r]: n_shards uint32 words of rank r,
 * zero-initialised, mapped here) runs before the first iteration and after each one, with epochs
 * epoch_base + 1 .. epoch_base + iterations + 1; every rank must call with the same arguments
 * (except rank, device, stream) and the caller advances epoch_base by iterations + 1 per call.
 * Same result as povs_shuffle_v1 on the concatenated deck with the same seed.
 * No reference counterpart (the reference has no multi-GPU code).
 */
#define POVS_MAX_SHARDS 8
#define POVS_DEV_PEER_TIMEOUT 4 /* device status bit: a peer GPU did not reach the barrier in time */
int povs_shuffle_sharded_v1(void* const* shard_ptrs, void* const* scratch_ptrs, const int64_t* shard_rows,
                            int32_t n_shards, int32_t rank, int64_t row_bytes, const int64_t* offsets,
                            int32_t n_offsets, int32_t iterations, int32_t pblock, int32_t vblock, uint64_t seed,
                            void* const* peer_flags, uint32_t epoch_base, int32_t device, void* stream,
                            uint32_t flags);

/*
 * Time limit of the cross-GPU barrier between iterations of povs_shuffle_sharded_v1 (process-wide;
 * 0 restores the default of 20 s).  A barrier that gives up sets POVS_DEV_PEER_TIMEOUT in the
 * device status word and returns, so the context stays usable.  No reference counterpart.
 */
int povs_set_peer_wait_limit_v1(uint64_t limit_ns);

/*
 * Let kernels on `device` read and write `peer`'s memory (cudaDeviceEnablePeerAccess; enabling it
 * twice is not an error).  Needed before povs_shuffle_shards_v1 gets shards on other GPUs of the
 * node.  No reference counterpart (the reference is single-GPU).
 */
int povs_enable_peer_access_v1(int32_t device, int32_t peer);

/*
 * Host only (no GPU needed): numpy.random.RandomState(seed).shuffle(arange(n)) into out[0 .. n-1],
 * the permutation the reference's NumPy path applies to a vblock of n rows under per-vblock seed
 * `seed` (src/povs/numpy.py:125-136).  The tables of the POVS_FLAG_REFERENCE_NUMPY mode are built
 * from it.
 */
int povs_numpy_path_perm_v1(uint32_t seed, int32_t n, int32_t* out);

/* CUDA IPC of device memory between the processes of a sharded deck (64-byte handles). */
int povs_ipc_export_v1(const void* ptr, int32_t device, void* handle_out, int64_t* offset_out);
int povs_ipc_import_v1(const void* handle, int64_t offset, int32_t device, void** ptr_out, void** base_out);
int povs_ipc_close_v1(void* base, int32_t device);

/* Read and clear the device status word of `device` (synchronizes the device's context). Writes bits to *status. */
int povs_device_status_v1(int32_t device, int32_t* status);

/* Free the per-device context (status word, cached graphs) of every device touched. */
int povs_release_v1(void);

/* Message describing the last error returned on the calling thread ("" if none). */
const char* povs_last_error_string(void);

/* Library version: major * 10000 + minor * 100 + patch. */
int32_t povs_version(void);

/*
 * Advanced: process-wide launch tuning (no reference counterpart; the reference
 * fixes these at compile time through template parameters, povs.cu:116,433-436).
 *   stage_cap   max bytes of one shared-memory data stage; vblocks whose V*P rows exceed it
 *               are processed in column slabs (default 32768)
 *   n_stages    max data stages in a CTA's ring, 2..16 (default 8; fewer when shared memory is short)
 *   movers      warps per CTA that copy rows (default 4)
 *   permuters   warps per CTA that compute members and permutations (default 4); movers + permuters <= 16
 *   force_plain 1 = plain vector loads instead of TMA bulk copies (whole rows of 4-byte multiples
 *               are then copied asynchronously); 2 = plain loads issued synchronously
 *   copy_bytes  target bytes of one bulk copy when whole rows are staged (default 8192)
 */
int povs_set_tuning_v1(int32_t stage_cap, int32_t n_stages, int32_t movers, int32_t permuters, int32_t force_plain,
                       int32_t copy_bytes);

/*
 * Advanced: largest packed unit, in bytes (process-wide; no reference counterpart).  Vblocks of
 * device-randomness in-place shuffles whose V*P rows are small travel several per unit (up to 32 / V
 * vblocks, 1024 rows and this many bytes per unit), so that per-unit costs are paid once for all of
 * them; the result is the same.  0 turns packing off; the default is 16384.
 */
int povs_set_pack_bytes_v1(int32_t pack_bytes);

/*
 * Advanced: report the launch plan povs_shuffle_v1 would use, as int64 values
 * {grid, block, dynamic smem, sort elements per lane, bulk (0/1), slab bytes, slabs,
 *  stages per CTA, stage bytes, vector bytes, vblocks, SM count, rows per bulk copy,
 *  permutation slots, mover warps, permuter warps, vblocks per unit, rows per unit,
 *  wide-row store kernel (0/1), chunked store kernel (0/1)}; returns how many were written.
 */
int povs_describe_plan_v1(void* data, int64_t n_rows, int64_t row_bytes, int32_t pblock, int32_t vblock,
                          int32_t device, int64_t* out, int32_t n_out);

/*
 * Advanced: the same plan computed on the host for given device resources, without a GPU: SM
 * count, the opt-in maximum of dynamic shared memory per block, shared memory per SM and threads
 * per SM (B200: 148, 232448, 233472, 2048).  data_address only sets the alignment the plan sees
 * (nonzero).  Same output as povs_describe_plan_v1, under the process-wide tuning.  For checking
 * plans in tests and tools; replaces nothing in the reference.
 */
int povs_plan_for_resources_v1(uint64_t data_address, int64_t n_rows, int64_t row_bytes, int32_t pblock,
                               int32_t vblock, int32_t sm_count, int32_t smem_optin, int32_t smem_per_sm,
                               int32_t max_threads_per_sm, int64_t* out, int32_t n_out);

/*
 * Allocation-free variant of povs_apply_v1 (no counterpart in the reference).
 *
 * For callers that cannot allocate GPU memory while they run - for example a process whose
 * memory pool has already reserved the GPU's free memory, or a service that forbids allocation
 * after start-up to keep its footprint fixed.  The injected randomness is passed in HOST memory
 * (same layouts as povs_apply_v1: assign_host int64 [iterations][n_v][V], perms_host int32
 * [iterations][n_v][V*P]) and staged, one iteration at a time, in a scratch array that is part
 * of the library image: POVS_STATIC_SCRATCH_BYTES of device memory that every GPU which loads
 * the library holds until the process exits.  The call allocates nothing (no cudaMalloc, no
 * CUDA graph); it launches the same kernels as povs_apply_v1 and gives the same bytes.
 *
 * Limit: one iteration needs 256 + round_up(8 * n_v * V, 256) + 4 * n_v * V * P bytes; larger
 * decks are rejected with POVS_ERR_UNSUPPORTED (use povs_apply_v1 then).
 * The first call on a device looks up the scratch array's device address (with that device
 * current) and reads its limits; make that first call before any stream capture.  With lazy
 * module loading (the CUDA 12 default) the array and the kernels come into being on the library's
 * first use on a device, so make one povs call there (iterations = 0 is enough: the set-up still
 * runs) before a memory pool reserves the GPU's free memory or the process stops allocating.
 * Every call shares the one array, which keeps the last call's contents (the status word in it is
 * cleared at the start of each call): calls that overlap on the GPU race.  Device failures (a
 * wait that timed out, an out-of-range injected permutation entry) are reported only with
 * POVS_FLAG_SYNC, the one flag accepted: the call then synchronizes `stream` and returns
 * POVS_ERR_DEVICE_STATUS; povs_device_status_v1 does not see this entry's status word.  Without it
 * the call returns after enqueueing, and the host arrays must stay unchanged until the stream has
 * run the work (pinned host memory is read asynchronously).
 */
#define POVS_STATIC_SCRATCH_BYTES (8u * 1024u * 1024u)
int povs_apply_static_v1(void* data, int64_t n_rows, int64_t row_bytes, int32_t pblock, int32_t vblock,
                         int32_t iterations, const int64_t* offsets_per_iter, const int64_t* assign_host,
                         const int32_t* perms_host, int32_t sort_members, int32_t device, void* stream,
                         uint32_t flags);

/*
 * Batched decks: n_decks independent decks of the same geometry, deck d at
 * data + d * deck_stride (bytes; deck_stride >= n_rows * row_bytes), all shuffled by one launch
 * per iteration.  Deck d ends exactly as povs_shuffle_v1 on it alone with seed seeds[d] would
 * leave it.  `seeds` is a DEVICE array of n_decks seeds that must stay unchanged until the stream
 * has run the work.  Flags as povs_shuffle_v1.
 * Replaces the reference's loop of one povs.shuffle call per episode in its bias exercises
 * (src/povs/eval/exercises.py:387-389, 247-249).
 */
int povs_shuffle_batch_v1(void* data, int64_t n_decks, int64_t deck_stride, int64_t n_rows, int64_t row_bytes,
                          const int64_t* offsets, int32_t n_offsets, int32_t iterations, int32_t pblock,
                          int32_t vblock, const uint64_t* seeds, int32_t device, void* stream, uint32_t flags);

/*
 * Travel-distance histogram over shuffled episodes (all pointers are device memory; asynchronous
 * on `stream`).  ids: int32 (id_bytes 4) or int64 (id_bytes 8); element i of episode e at
 * ids[e * episode_stride + i * element_stride], each episode a permutation of 0 .. deck-1.
 * kind 0: counts[(i - v) mod deck] += 1 for every element (positional travel distance,
 * get_tvd, src/povs/eval/metrics.py:38-87).  kind 1: counts[((v[(i + step) mod deck] - v[i]) - step)
 * mod deck] += 1 for every position (2-gram relative travel distance with step = skip + 1,
 * get_ngram_tvd with n = 2, metrics.py:147-172).  counts: deck uint64 bins, ADDED to.
 */
int povs_travel_histogram_v1(const void* ids, int32_t id_bytes, int64_t n_episodes, int64_t deck,
                             int64_t episode_stride, int64_t element_stride, int32_t kind, int64_t step,
                             uint64_t* counts, int32_t device, void* stream);

/*
 * n-gram keys (n >= 2) over shuffled episodes, for the sparse n-gram TVD (get_ngram_tvd with
 * n > 2, metrics.py:173-248): for every episode e and anchor a (positions[j] for j < n_positions,
 * or every position 0 .. deck-1 when positions is NULL), keys[e * count + j] =
 * sum over k = 1 .. n-1 of (((v[(a + k*step) mod deck] - v[a]) - k*step) mod deck) * deck^(n-1-k),
 * in wrapping 64-bit arithmetic.  Same id layout as povs_travel_histogram_v1.
 */
int povs_ngram_keys_v1(const void* ids, int32_t id_bytes, int64_t n_episodes, int64_t deck, int64_t episode_stride,
                       int64_t element_stride, int32_t n, int64_t step, const int64_t* positions,
                       int64_t n_positions, int64_t* keys, int32_t device, void* stream);

/*
 * The distinct n-gram keys of povs_ngram_keys_v1 (same arguments) counted without sorting, for the
 * sparse n-gram TVD (metrics.py:173-248, which sorts the keys with np.unique): an open-addressing
 * hash table in `table` (device, 2 * slots + 1 uint64, overwritten; slots a power of two above the
 * number of keys, twice it or more keeps probes short), then the multiplicities of the counts:
 * mult[c] (device, mult_bins uint64, overwritten) = distinct keys seen exactly c times for
 * 1 <= c < mult_bins, mult[0] = distinct keys seen mult_bins times or more, whose counts go to
 * overflow[0 .. min(mult[0], overflow_cap) - 1] (device, any order).  The TVD needs only these:
 * observed keys = sum of mult, and sum over keys of |count / observations - p_ref|.  A key that
 * finds no free slot sets POVS_DEV_TABLE_FULL in the device status word.  No reference
 * counterpart as an entry point (the reference counts on the host).
 */
#define POVS_DEV_TABLE_FULL 8
int povs_ngram_count_v1(const void* ids, int32_t id_bytes, int64_t n_episodes, int64_t deck, int64_t episode_stride,
                        int64_t element_stride, int32_t n, int64_t step, const int64_t* positions,
                        int64_t n_positions, uint64_t* table, int64_t slots, uint64_t* mult, int64_t mult_bins,
                        uint64_t* overflow, int64_t overflow_cap, int32_t device, void* stream);

/*
 * Row operators whose order follows from scores.  Every pointer is a multiple of its elements' size
 * (others are refused).  Element types of scores and rows: */
#define POVS_FLOAT32 0
#define POVS_BFLOAT16 1
#define POVS_FLOAT16 2

/*
 * Draw one id per row from scores (all pointers are device memory; asynchronous on `stream`).
 * Row r has the scores logits[r * row_stride + i], 0 <= i < width (strides in elements), and the
 * number uniforms[r] (float or double: uniform_bytes 4 or 8; taken into [0, 1)).  NaN and -infinity
 * are never drawn.  With the weights w_i = exp((x_i - max x) / temperature) and the ids in
 * descending order of their score, equal scores by the lowest id:
 *   top_k > 0   keeps the first top_k ids;
 *   top_p < 1   keeps, of those, each id before which the kept weights sum to less than top_p of
 *               their whole sum (the first always);
 *   min_p > 0   keeps, of those, the ids with w_i >= min_p (the highest score's always).
 * ids[r] is the lowest id at which the kept weights, summed in id order, exceed uniforms[r] of their
 * whole sum.  temperature 0 (in the array: any value not above 0, or NaN): the lowest id of the
 * highest score.  Where some scores are +infinity, they alone have a weight, each the same.  A row without a
 * number above -infinity gets -1.  temperatures, top_ks, top_ps and min_ps are NULL or hold one value
 * per row in place of the value beside them; temperatures above 1e28 count as 1e28, those below 1e-36 as
 * 1e-36.  Weights and sums have 64 bits, good to 2^-40 of the row's sum.  Where top_p keeps, or top_k with top_p
 * reaches, more ids than fit a list of 2048, top_p's border may be found from weights rounded to whole numbers
 * that keep a row's sum below 2^63: with n = ceil(log2(width)) good to 2^(2n - 63) of the sum at worst (2^-29 for
 * 131072 ids).  uniforms 0 draws the first id with any weight.  The id is the same on every run.
 * No reference counterpart: numpy.random.Generator.choice beside its Generator.shuffle baseline.
 */
int povs_sample_v1(const void* logits, int32_t dtype, int64_t rows, int64_t width, int64_t row_stride,
                   const void* uniforms, int32_t uniform_bytes, const float* temperatures, double temperature,
                   const int32_t* top_ks, int64_t top_k, const float* top_ps, double top_p, const float* min_ps,
                   double min_p, int64_t* ids, int32_t device, void* stream);

/*
 * Choose top_k experts for every row from its scores (device memory; asynchronous on `stream`).
 * Scores s = softmax or sigmoid of the row's logits; choice scores c = s + bias (bias: n_experts
 * floats or NULL; it moves the choice and not the weights).  With top_groups < n_groups, the experts
 * form n_groups groups of n_experts / n_groups neighbours; a group scores the sum of its two highest
 * choice scores (POVS_GROUP_TOP2) or its highest (POVS_GROUP_MAX), and only the top_groups best
 * groups' experts can be chosen.  experts[r * top_k + j]: the j-th highest c, equal ones by the lowest
 * index; weights[r * top_k + j] = scale * s of it, divided by the sum of the row's chosen s with
 * renormalize (also where those are too small for 32 bits).  Without bias and groups the order is the logits'; else choices are made on scores
 * computed in 64 bits.  An expert whose logit or choice
 * score is -infinity is never chosen; a row with fewer than top_k others ends with experts -1 of
 * weight 0.  A NaN score ranks below every number.  No reference counterpart.
 */
#define POVS_SCORE_SOFTMAX 0
#define POVS_SCORE_SIGMOID 1
#define POVS_GROUP_TOP2 0
#define POVS_GROUP_MAX 1
#define POVS_MAX_ROUTE_EXPERTS 1024
#define POVS_MAX_TOP_K 32
int povs_route_v1(const void* logits, int32_t dtype, int64_t rows, int32_t n_experts, int64_t row_stride,
                  const float* bias, int32_t top_k, int32_t scoring, int32_t n_groups, int32_t top_groups,
                  int32_t group_score, int32_t renormalize, float scale, int32_t* experts, float* weights,
                  int32_t device, void* stream);

/* Gradient of povs_route_v1's weights: grad_logits (rows, n_experts), contiguous, of the logits'
 * type, from `experts` as povs_route_v1 wrote them and grad_weights (rows, top_k). */
int povs_route_backward_v1(const void* logits, int32_t dtype, int64_t rows, int32_t n_experts, int64_t row_stride,
                           int32_t top_k, int32_t scoring, int32_t renormalize, float scale, const int32_t* experts,
                           const float* grad_weights, void* grad_logits, int32_t device, void* stream);

/*
 * The order that brings rows with the same expert together (device memory; asynchronous on
 * `stream`): a stable counting sort of n_entries = rows * top_k expert numbers (int32 or int64:
 * id_bytes 4 or 8).  slots[i]: the place of entry i, sources[slot]: the entry there, offsets[e]: the
 * first slot of expert e (n_experts + 1 numbers).  Within an expert, entries keep their order.  An
 * entry outside 0 .. n_experts-1 (-1 by convention) takes no slot: slots -1, and as many sources at
 * the end are -1.  `workspace` (device) holds povs_plan_rows_workspace_v1 bytes (NULL where that is
 * 0) and belongs to the call until the stream has run it.  No reference counterpart.
 */
#define POVS_MAX_PLAN_EXPERTS 4096
int64_t povs_plan_rows_workspace_v1(int64_t n_entries, int32_t n_experts);
int povs_plan_rows_v1(const void* experts, int32_t id_bytes, int64_t n_entries, int32_t n_experts, int32_t* slots,
                      int32_t* sources, int32_t* offsets, void* workspace, int64_t workspace_bytes, int32_t device,
                      void* stream);

/*
 * Copy rows to their slots (device memory; asynchronous on `stream`): row r (row_bytes opaque bytes
 * at data + r * row_stride, bytes) to out + slot * row_bytes for each of slots[r * top_k ..
 * + top_k - 1] in 0 .. n_slots-1.  The rows of `out` from *used (device) on are zeroed.  Slots as
 * povs_plan_rows_v1 writes them name each place below *used once; with others, a place named twice holds pieces of
 * either row, and one named by none is left as it was.  `out` must not overlap `data`.  No reference counterpart (its moves
 * are in place).
 */
int povs_dispatch_rows_v1(const void* data, int64_t rows, int64_t row_bytes, int64_t row_stride,
                          const int32_t* slots, int32_t top_k, const int32_t* used, void* out, int64_t n_slots,
                          int32_t device, void* stream);

/*
 * Weighted sums of slots (device memory; asynchronous on `stream`): out[r] = sum over j of
 * weights[r * top_k + j] * data[slots[r * top_k + j]] (weights NULL: ones), summed in 32 bits in the
 * order of j and rounded once.  data: n_slots rows of `width` elements, data_stride elements apart;
 * out: contiguous.  Slots outside 0 .. n_slots-1 are left out; a row without a slot is 0.
 * No reference counterpart.
 */
int povs_combine_rows_v1(const void* data, int32_t dtype, int64_t n_slots, int64_t width, int64_t data_stride,
                         const int32_t* slots, int64_t rows, int32_t top_k, const float* weights, void* out,
                         int32_t device, void* stream);

/* Gradients of povs_combine_rows_v1 from grad (rows, width), contiguous: grad_data (n_slots, width),
 * contiguous, or NULL, where the slots from *used on are zeroed (each place below is named once, as by
 * povs_plan_rows_v1); grad_weights (rows, top_k), or NULL, for which alone `data` is read. */
int povs_combine_backward_v1(const void* grad, const void* data, int32_t dtype, int64_t n_slots, int64_t width,
                             int64_t data_stride, const int32_t* slots, int64_t rows, int32_t top_k,
                             const float* weights, const int32_t* used, void* grad_data, float* grad_weights,
                             int32_t device, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* POVS_H */
