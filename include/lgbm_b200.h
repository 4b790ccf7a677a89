/*
 * lgbm_b200 — C ABI of the B200 histogram tree learner.
 *
 * This ABI replaces the reference's compute seam, `trait Backend` of
 * BectorVoom/lightgbm_rs (crates/lgbm-compute/src/lib.rs:1092-2782), and the
 * whole-tree / whole-iteration device paths behind it. Each entry point names
 * the reference interface it stands in for.
 *
 * Conventions
 *  - Every function returns an int status (LGBM_B200_*). On failure,
 *    lgbm_b200_last_error() returns a thread-local message. No C++ exception,
 *    abort or device trap crosses this boundary.
 *  - Host pointers are borrowed for the duration of the call only.
 *  - Device state is owned by opaque handles with create/destroy pairs.
 *  - Histograms are interleaved [g0, h0, g1, h1, ...] f64 cells, as in the
 *    reference (GET_GRAD(i) = hist[2i], GET_HESS(i) = hist[2i+1]).
 */
#ifndef LGBM_B200_H
#define LGBM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. 1..5 mirror lgbm_compute::error::ComputeError
 * (crates/lgbm-compute/src/error.rs:19-80). */
#define LGBM_B200_OK 0
#define LGBM_B200_BIN_OUT_OF_RANGE 1
#define LGBM_B200_LENGTH_MISMATCH 2
#define LGBM_B200_CAPABILITY_UNAVAILABLE 3
#define LGBM_B200_RUNTIME 4
#define LGBM_B200_NON_FINITE 5
#define LGBM_B200_INVALID_ARGUMENT 6

/* Missing-value handling of a feature (lgbm-dataset/src/bin_mapper.rs:15-20). */
#define LGBM_B200_MISSING_NONE 0
#define LGBM_B200_MISSING_ZERO 1
#define LGBM_B200_MISSING_NAN 2

/* Objectives on the path (lgbm-objective/src/binary.rs, regression.rs, rank.rs). */
#define LGBM_B200_OBJECTIVE_BINARY 0
#define LGBM_B200_OBJECTIVE_L2 1
#define LGBM_B200_OBJECTIVE_LAMBDARANK 2

/* Largest query a lambdarank objective accepts: the DCG discount table's length
 * (K_MAX_POSITION, lgbm-metric/src/dcg_calculator.rs:32). */
#define LGBM_B200_MAX_QUERY_ROWS 10000

/* Gradient-pair encodings accepted by lgbm_b200_learner_grow_tree. */
#define LGBM_B200_GH_F32 0       /* float g[N], float h[N] */
#define LGBM_B200_GH_INT8_PAIR 1 /* int8 (qg, qh) per row + grad/hess scales */

/* lgbm_compute::gain::GainConfig (crates/lgbm-compute/src/gain.rs:904-960). */
typedef struct lgbm_b200_gain_config {
  int32_t min_data_in_leaf;
  int32_t _reserved;
  double min_sum_hessian_in_leaf;
  double max_delta_step;
  double lambda_l1;
  double lambda_l2;
  double min_gain_to_split;
  double path_smooth;
  double parent_output;
  /* categorical splits (feature_histogram_categorical.rs; LightGBM defaults 100, 32,
   * 4, 10, 10) */
  int32_t min_data_per_group;
  int32_t max_cat_threshold;
  int32_t max_cat_to_onehot;
  int32_t _reserved2;
  double cat_l2;
  double cat_smooth;
} lgbm_b200_gain_config;

/* lgbm_compute::gain::SplitInfo (crates/lgbm-compute/src/gain.rs:1040-1065).
 * gain == -inf means "no split". */
typedef struct lgbm_b200_split_info {
  uint32_t threshold;
  int32_t default_left;
  int32_t left_count;
  int32_t right_count;
  double gain;
  double left_sum_gradient;
  double left_sum_hessian;
  double right_sum_gradient;
  double right_sum_hessian;
  double left_output;
  double right_output;
} lgbm_b200_split_info;

/* The per-feature fields of lgbm_treelearner::FeatureColumn the learner reads
 * (crates/lgbm-treelearner/src/learner.rs:87-140). offset is derived:
 * 1 iff most_freq_bin == 0 (crates/lgbm-treelearner/src/lib.rs:89-95). */
typedef struct lgbm_b200_feature_meta {
  int32_t num_bin;
  int32_t default_bin;
  int32_t most_freq_bin;
  int32_t missing_type;
  int32_t bin_type; /* 0 numerical, 1 categorical (BinType, bin_mapper.rs:22-26) */
} lgbm_b200_feature_meta;

/* lgbm_compute::BatchedSplitFeature (crates/lgbm-compute/src/kernels/split.rs:77). */
typedef struct lgbm_b200_batched_feature {
  int64_t slot_off;
  uint32_t num_bin;
  int32_t offset;
  uint32_t default_bin;
  uint32_t most_freq_bin;
  int32_t skip_default_bin;
  int32_t na_as_missing;
  int32_t run_forward;
  int32_t _reserved;
} lgbm_b200_batched_feature;

/* Tree node arrays (crates/lgbm-model/src/tree.rs:94-160). Caller-owned host
 * arrays sized for max_leaves leaves / max_leaves-1 internal nodes. */
typedef struct lgbm_b200_tree {
  int32_t num_leaves;
  int32_t max_leaves;
  int32_t* left_child;
  int32_t* right_child;
  int32_t* split_feature;
  uint32_t* threshold_bin;
  float* split_gain;
  int8_t* decision_type;
  double* leaf_value;
  double* leaf_weight;
  int32_t* leaf_count;
  double* internal_value;
  int32_t* internal_count;
  /* per internal node, 8 words: the set of bins a categorical node sends left
   * (decision_type bit 0; threshold_bin is the categorical-node index); may be
   * NULL. The category bitsets of the model text follow from the feature's
   * bin_to_category (Tree::split_categorical, lgbm-model/src/tree.rs:710-770). */
  uint32_t* cat_bins;
} lgbm_b200_tree;

/* SerialTreeLearner construction parameters
 * (crates/lgbm-treelearner/src/learner.rs:627). */
typedef struct lgbm_b200_learner_config {
  int32_t num_leaves;
  int32_t max_depth;
  lgbm_b200_gain_config gain;
} lgbm_b200_learner_config;

/* The Gbdt training knobs the path reads (crates/lgbm-boosting/src/gbdt.rs:691-1300). */
typedef struct lgbm_b200_train_config {
  lgbm_b200_learner_config learner;
  int32_t objective;
  int32_t use_quantized_grad;
  int32_t num_grad_quant_bins;
  int32_t boost_from_average;
  double sigmoid;
  double learning_rate;
  /* Lambdarank only (Lambdarank::new, lgbm-objective/src/rank.rs:152-227): the query
   * boundaries of this device's rows (num_queries + 1 ascending prefix sums from 0 to
   * num_data; borrowed for the call), lambdarank_truncation_level, lambdarank_norm,
   * and the label gains (num_label_gain = 0: the default 2^i - 1 for i < 31). A
   * ranking objective has no boost-from-average score. */
  const int32_t* query_boundaries;
  int32_t num_queries;
  int32_t lambdarank_truncation_level;
  int32_t lambdarank_norm;
  int32_t num_label_gain;
  const double* label_gain;
  /* use_quantized_grad only: stochastic rounding (the reference's default,
   * crates/lgbm-core/src/config/mod.rs:485): rounding offsets from the reference's
   * seeded xorshift64 (crates/lgbm-treelearner/src/gradient_discretizer.rs:252-262),
   * seed ((iteration << 20) ^ 0x51702010) per iteration (crates/lgbm-boosting/src/
   * gbdt.rs:950), drawn over the rows of the whole job in row order (a data-parallel
   * job: rank 0's rows first). 0: deterministic rounding (offset 0.5). */
  int32_t stochastic_rounding;
  int32_t _reserved0;
} lgbm_b200_train_config;

/* BinMapper::find_bin_from_column parameters (crates/lgbm-dataset/src/bin_mapper.rs:642-675). */
typedef struct lgbm_b200_bin_config {
  int32_t max_bin;
  int32_t min_data_in_bin;
  int32_t min_data_in_leaf;
  int32_t pre_filter;
  int32_t use_missing;
  int32_t zero_as_missing;
  int32_t bin_construct_sample_cnt;
  int32_t data_random_seed;
} lgbm_b200_bin_config;

/* BinMapper result fields (crates/lgbm-dataset/src/bin_mapper.rs:45-60). */
typedef struct lgbm_b200_bin_mapper {
  int32_t num_bin;
  int32_t missing_type;
  int32_t default_bin;
  int32_t most_freq_bin;
  int32_t is_trivial;
  int32_t _reserved;
  double min_val;
  double max_val;
  double sparse_rate;
} lgbm_b200_bin_mapper;

typedef struct lgbm_b200_dataset lgbm_b200_dataset;
typedef struct lgbm_b200_learner lgbm_b200_learner;
typedef struct lgbm_b200_booster lgbm_b200_booster;

/* Thread-local message of the last failed call on this thread ("" if none). */
const char* lgbm_b200_last_error(void);

/* ABI version of this header (major * 100 + minor). */
int32_t lgbm_b200_abi_version(void);

/* Number of CUDA devices visible (0 when none; never an error). */
int lgbm_b200_device_count(int32_t* out);

/* Frees the device blocks (1 MB and larger) that destroyed datasets and
 * boosters left in this library's per-process cache, on `device` (-1: every
 * device), and reports the bytes freed (may be NULL). No counterpart in the
 * reference, whose CubeCL runtime keeps its own memory pool. The cache is
 * also trimmed on its own before a cudaMalloc is reported as failed. */
int lgbm_b200_release_cached_memory(int32_t device, int64_t* released_bytes);

/* ------------------------------------------------------------------ binning */

/* BinMapper::find_bin_from_column + value_to_bin
 * (crates/lgbm-dataset/src/bin_mapper.rs:642-675, :148-199, :201-415).
 * upper_bounds receives num_bin values (capacity upper_cap); bins_out (may be
 * NULL) receives value_to_bin of every row. Host-only; needs no GPU. */
int lgbm_b200_bin_column(const double* column, int64_t n, const lgbm_b200_bin_config* cfg,
                         lgbm_b200_bin_mapper* mapper_out, double* upper_bounds,
                         int32_t upper_cap, uint32_t* bins_out);

/* BinMapper::find_bin_categorical + value_to_bin for a categorical column
 * (crates/lgbm-dataset/src/bin_mapper.rs:416-641, :148-199): categories by
 * descending count, bin 0 the dummy bin of NaN / negative / unseen values.
 * bin_to_category receives num_bin category values (bin 0: -1; capacity cap);
 * mapper_out->_reserved is 1 (categorical). Host-only; needs no GPU. */
int lgbm_b200_bin_column_categorical(const double* column, int64_t n,
                                     const lgbm_b200_bin_config* cfg,
                                     lgbm_b200_bin_mapper* mapper_out, int32_t* bin_to_category,
                                     int32_t cap, uint32_t* bins_out);

/* BinMapper::find_bin_from_column of many numerical columns at once, on the device
 * (crates/lgbm-dataset/src/bin_mapper.rs:642-675 with find_bin_numeric :201-415): every
 * column's sample (the same rows for every column: create_sample_indices, :92-95) is
 * gathered on the host, then sorted and binned on the device; the mappers and bounds
 * equal lgbm_b200_bin_column's. columns: feature-major host arrays of n f32
 * (value_width 4) or f64 (8) values. mappers_out[f] and upper_bounds[f * upper_cap ...]
 * (num_bin values; upper_cap >= max_bin + 2) receive the results. Categorical columns
 * go through lgbm_b200_bin_column_categorical. */
int lgbm_b200_find_bins(int32_t device, const void* const* columns, int32_t value_width,
                        int64_t n, int32_t num_features, const lgbm_b200_bin_config* cfg,
                        lgbm_b200_bin_mapper* mappers_out, double* upper_bounds,
                        int32_t upper_cap);

/* ------------------------------------------------------ per-op Backend mirror */

/* Backend::construct_histograms (crates/lgbm-compute/src/lib.rs:1119-1126):
 * histogram of one feature over all rows. out has 2*num_bin cells.
 * f32 g/h accumulate in 64-bit fixed point (relative error ~1e-11 of the
 * reference's f64 fold). num_bin <= 256. */
int lgbm_b200_construct_histograms(const uint32_t* binned, const float* gradients,
                                   const float* hessians, int64_t n, uint32_t num_bin,
                                   double* out);

/* Backend::find_best_split (crates/lgbm-compute/src/lib.rs:1174-1189), computed
 * by the device threshold-scan kernel; bit-exact with the reference CPU scan. */
int lgbm_b200_find_best_split(const double* hist, const lgbm_b200_gain_config* cfg,
                              uint32_t num_bin, int32_t offset, uint32_t default_bin,
                              uint32_t most_freq_bin, int32_t skip_default_bin,
                              int32_t na_as_missing, int32_t run_forward, double sum_gradient,
                              double sum_hessian, int32_t num_data, lgbm_b200_split_info* out);

/* Backend::find_best_splits_batched (crates/lgbm-compute/src/lib.rs:1500-1509). */
int lgbm_b200_find_best_splits_batched(const double* buf, int64_t buf_len,
                                       const lgbm_b200_batched_feature* feats, int32_t n_feats,
                                       const lgbm_b200_gain_config* cfg, double sum_gradient,
                                       double sum_hessian, int32_t num_data,
                                       lgbm_b200_split_info* out);

/* Backend::data_partition (crates/lgbm-compute/src/lib.rs:1206-1215): stable
 * partition of rows 0..n-1; order_out = [left ascending | right ascending]. */
int lgbm_b200_data_partition(const uint32_t* bins, int64_t n, uint32_t num_bin, uint32_t min_bin,
                             uint32_t max_bin, uint32_t threshold, uint32_t most_freq_bin,
                             uint32_t* order_out, int64_t* split_point_out);

/* The kernel-level partition with the whole missing-value routing fan-out:
 * partition_leaf_stable / partition_on_device (crates/lgbm-compute/src/kernels/
 * data_partition.rs:487-520, routing RouteFlags::derive + route_to_left :325-406,
 * :64-138). Arguments as lgbm_b200_data_partition plus default_bin, missing_type
 * (0 None, 1 Zero, 2 NaN) and default_left. missing_type 1 routes the zero bin
 * (min_bin + default_bin - [most_freq_bin == 0]) and 2 the NA bin (max_bin) by
 * default_left, unless the most frequent bin is that bin; min_bin == max_bin is the
 * degenerate one-bin feature. Host buffers; result [left ascending | right
 * ascending]. */
int lgbm_b200_data_partition_missing(const uint32_t* bins, int64_t n, uint32_t num_bin,
                                     uint32_t min_bin, uint32_t max_bin, uint32_t threshold,
                                     uint32_t most_freq_bin, uint32_t default_bin,
                                     int32_t missing_type, int32_t default_left,
                                     uint32_t* order_out, int64_t* split_point_out);

/* Allocation-free variant of lgbm_b200_data_partition. No counterpart in the
 * reference: it exists for callers that cannot call cudaMalloc when they
 * partition rows. Examples are a host engine whose device memory belongs to its
 * own pool allocator, which has reserved the HBM up front so that a cudaMalloc
 * can fail or fragment its reservation, and a latency-bound loop that cannot
 * pay for cudaMalloc/cudaFree, which synchronise the whole device.
 *
 * Same argument meaning and result as lgbm_b200_data_partition, except that
 * `bins` (n bytes, one bin per row), `order_out` (n words) and
 * `split_point_out` (one int64) are DEVICE pointers on the current device, and
 * the work is enqueued on `stream` (a cudaStream_t; NULL is the legacy default
 * stream) without waiting for it: the outputs are ready once the stream
 * reaches that point. Bins are not range-checked on this path; a bin outside
 * [min_bin, max_bin] goes where the most frequent bin goes.
 *
 * Scratch: the partition's look-back status words (one per 2048-row tile), two
 * counters and the routing descriptor live in a fixed array compiled into the
 * library, one per device, 256 B + 8 B per tile = 262,400 B at the limit. The
 * function allocates nothing. n above LGBM_B200_NOALLOC_MAX_ROWS fails with
 * LGBM_B200_CAPABILITY_UNAVAILABLE and enqueues no work. Each call first
 * clears, on `stream`, the status words and counters it uses; they must start
 * at zero. Every call on a device shares the one array, so calls that overlap
 * on the GPU (different streams, or different host threads) race and return
 * wrong results: serialise them. The first call on each device looks the
 * array up with cudaGetSymbolAddress (with that device current); make that
 * first call before any stream capture. A failed lookup returns
 * LGBM_B200_RUNTIME and is tried again by the next call.
 *
 * The partition's look-back waits are bounded. If one runs out (a tile whose
 * predecessor never published, e.g. under heavy preemption), `order_out` is
 * left incomplete and *split_point_out is set to the sentinel -1 on the
 * stream: check it before using the order. The allocating entry point
 * returns LGBM_B200_RUNTIME in the same case. */
#define LGBM_B200_NOALLOC_MAX_ROWS 67108864 /* 2^26 rows */
int lgbm_b200_data_partition_noalloc(const uint8_t* bins, int64_t n, uint32_t num_bin,
                                     uint32_t min_bin, uint32_t max_bin, uint32_t threshold,
                                     uint32_t most_freq_bin, uint32_t* order_out,
                                     int64_t* split_point_out, void* stream);

/* Backend::subtract_histograms (crates/lgbm-compute/src/lib.rs:1314-1319). */
int lgbm_b200_subtract_histograms(const double* parent, const double* child, int64_t len,
                                  double* out);

/* ---------------------------------------------------- device-resident dataset */

/* Backend::upload_resident_bins (crates/lgbm-compute/src/lib.rs:1564): take
 * feature-major bin columns (bin_width 1, 2 or 4 bytes per bin) and keep a
 * row-major u8 bin matrix resident on `device`. Validates bin < num_bin once
 * (the learner's bin-range gate, learner.rs:1161-1187). */
int lgbm_b200_dataset_create(int32_t device, const void* const* columns, int32_t bin_width,
                             int64_t num_data, int32_t num_features,
                             const lgbm_b200_feature_meta* meta, lgbm_b200_dataset** out);
int lgbm_b200_dataset_destroy(lgbm_b200_dataset* ds);

/* The device dataset from raw feature values: BinMapper::value_to_bin
 * (crates/lgbm-dataset/src/bin_mapper.rs:148-199) runs on the device with the mappers
 * found on the host from each column's sample (lgbm_b200_bin_column /
 * lgbm_b200_bin_column_categorical with bins_out = NULL). columns: feature-major host
 * arrays of f32 (value_width 4) or f64 (8). upper_bounds[f] (numerical features) and
 * bin_to_category[f] (categorical features) hold num_bin values each. Replaces the
 * host binning loop of the reference's dataset construction
 * (crates/lgbm/src/booster.rs:381-540). */
int lgbm_b200_dataset_create_from_values(int32_t device, const void* const* columns,
                                         int32_t value_width, int64_t num_data,
                                         int32_t num_features,
                                         const lgbm_b200_feature_meta* meta,
                                         const double* const* upper_bounds,
                                         const int32_t* const* bin_to_category,
                                         lgbm_b200_dataset** out);
/* Copies the device bin matrix back: row-major u8 [num_data][stride], stride =
 * num_features rounded up to a multiple of 16. */
int lgbm_b200_dataset_copy_bins(const lgbm_b200_dataset* ds, uint8_t* out);
int lgbm_b200_dataset_num_data(const lgbm_b200_dataset* ds, int64_t* out);

/* ------------------------------------------------------------ tree learner */

/* SerialTreeLearner::new (crates/lgbm-treelearner/src/learner.rs:627). */
int lgbm_b200_learner_create(lgbm_b200_dataset* ds, const lgbm_b200_learner_config* cfg,
                             lgbm_b200_learner** out);
int lgbm_b200_learner_destroy(lgbm_b200_learner* learner);

/* Backend::grow_tree_on_device_with_cfg (crates/lgbm-compute/src/lib.rs:2771-2781):
 * grow one tree from host gradients. gh_kind LGBM_B200_GH_F32: gh = float[2][N]
 * (g then h); LGBM_B200_GH_INT8_PAIR: gh = int8 (qg, qh) per row and
 * quant_scales = {grad_scale, hess_scale, is_constant_hessian, num_grad_quant_bins}
 * as produced by GradientDiscretizer (gradient_discretizer.rs:145-191), in which
 * case the tree is bit-identical to the reference learner on the dequantized
 * gradients. indices_out (N), leaf_begin_out / leaf_count_out (num_leaves) may
 * be NULL; rows inside a leaf are a permutation of the reference's order. */
int lgbm_b200_learner_grow_tree(lgbm_b200_learner* learner, int32_t gh_kind, const void* gh,
                                const double* quant_scales, lgbm_b200_tree* tree_out,
                                uint32_t* indices_out, int32_t* leaf_begin_out,
                                int32_t* leaf_count_out);

/* ------------------------------------------------------------------ booster */

/* Gbdt (crates/lgbm-boosting/src/gbdt.rs:691-1300) with the score kept resident:
 * gradients, quantization, tree growth, shrinkage and score update all run on
 * the device; labels are copied once. */
int lgbm_b200_booster_create(lgbm_b200_dataset* ds, const float* labels,
                             const lgbm_b200_train_config* cfg, lgbm_b200_booster** out);
int lgbm_b200_booster_destroy(lgbm_b200_booster* b);
/* Run up to num_iterations boosting iterations; *done_out receives how many
 * produced a tree before training stopped (a 1-leaf tree after the first). */
int lgbm_b200_booster_train(lgbm_b200_booster* b, int32_t num_iterations, int32_t* done_out);
int lgbm_b200_booster_num_trees(const lgbm_b200_booster* b, int32_t* out);
/* Trees after shrinkage; the init score of boost_from_average is reported separately. */
int lgbm_b200_booster_get_tree(lgbm_b200_booster* b, int32_t index, lgbm_b200_tree* out);
int lgbm_b200_booster_init_score(const lgbm_b200_booster* b, double* out);
int lgbm_b200_booster_get_scores(lgbm_b200_booster* b, double* out);
/* The gradients of the most recent iteration (f32, before quantization). */
int lgbm_b200_booster_get_gradients(lgbm_b200_booster* b, float* g, float* h);
/* Device time of the last lgbm_b200_booster_train call in ms (out3[1]; the other
 * two entries are 0). */
int lgbm_b200_booster_phase_ms(const lgbm_b200_booster* b, double* out3);
/* Run ONE more boosting iteration outside the CUDA graph with CUDA events around
 * every kernel launch. ms_out[7] receives the summed device time per kernel class
 * {prepare, histogram build, fix+scan, partition, tree init, gradients, finish};
 * counts_out[8] = {kernel launches, histogram builds, rows streamed by the builds,
 * splits, parent rows streamed by the partitions, 1 if the partition kernel also
 * builds the child histogram, look-ahead partitions run, look-ahead partitions whose
 * leaf was the next split}. Builds and rows count the partitions whose result the tree
 * used. The iteration counts as a normal boosting iteration. */
int lgbm_b200_booster_profile_iteration(lgbm_b200_booster* b, double* ms_out,
                                        int64_t* counts_out);
/* Run `iterations` more boosting iterations through a CUDA graph of the same launch
 * sequence as lgbm_b200_booster_train (look-ahead stream included), whose tree kernels
 * stamp their device-time spans (%globaltimer at each CTA's entry and exit): a span is
 * first entry to last exit of one launch, as it ran in the pipeline. span_ms_out[7]
 * receives the mean per iteration of the summed spans per kernel class (same order as
 * profile_iteration; partition = the main-stream partitions). iter_ms_out[2] = {mean
 * device ms per iteration, mean summed spans of the look-ahead partitions, which run
 * beside the control steps}. counts_out[10] receives the same eight counters as
 * profile_iteration, summed over the iterations (counts_out[0]: stamped tree-kernel
 * launches), then the parent rows of the main partitions that ran inside control steps
 * (one device: a control step partitions the previous split's leaf itself when the
 * look-ahead did not) and the rows their child builds accumulated. No counterpart in the
 * reference (a profiling aid). */
int lgbm_b200_booster_profile_pipeline(lgbm_b200_booster* b, int32_t iterations,
                                       double* span_ms_out, double* iter_ms_out,
                                       int64_t* counts_out);
/* The raw spans of the last iteration lgbm_b200_booster_profile_pipeline ran: per slot
 * (0: the root build; 1 + 4*s + kind for split step s, kind 0 control step, 1 main-stream
 * partition, 2 look-ahead partition, 3 separate build) the earliest CTA entry and latest
 * CTA exit in %globaltimer ns; a slot not launched holds start = UINT64_MAX. phase_out
 * (optional, cap * 20 entries): for split step s, twenty marks at phase_out[20*s] (latest
 * CTA time, 0 when not reached). Eight control-step marks: pending split applied, feature
 * cells loaded, FixHistogram and child stores done, scans done, every feature of the CTA
 * done, pick inputs staged, pick made, control block written. Then six marks of the
 * step's look-ahead partition and six of its main partition, raised by the CTAs that hold
 * a tile: entry, setup done, first tile's rows routed, its prefix known, last tile
 * written, histogram flushed. *n_out receives the slot
 * count; at most cap entries of each span array are written. No counterpart in the
 * reference (a profiling aid). */
int lgbm_b200_booster_profile_spans(const lgbm_b200_booster* b, int32_t cap,
                                    uint64_t* start_out, uint64_t* end_out, uint64_t* phase_out,
                                    int32_t* n_out);
/* The launches timed by the last lgbm_b200_booster_profile_iteration, in launch order:
 * kernel class (the ms_out order of that call) and device ms of each timed span; *n_out
 * receives the count, at most cap entries are written. */
int lgbm_b200_booster_profile_launches(const lgbm_b200_booster* b, int32_t cap,
                                       int32_t* class_out, float* ms_out, int32_t* n_out);

/* ---------------------------------------------------- data-parallel training */

/* Several GPUs train one model on a dataset sharded by rows, one process (or
 * thread) per GPU: LightGBM's data-parallel tree learner. The reference has no
 * counterpart: it maps tree_learner=data/feature/voting back to serial
 * (crates/lgbm-core/src/config/set.rs:592-600). Every rank keeps its own rows;
 * after each histogram build the ranks sum the integer child histogram and its
 * left-row count over NCCL (one all-reduce per split), so all ranks take the
 * same decisions and hold the same trees. With quantized gradients the trees
 * are bit-identical to single-GPU training on all rows.
 *
 * NCCL is loaded at run time (libnccl.so.2); without it these calls return
 * LGBM_B200_CAPABILITY_UNAVAILABLE. Rank 0 makes the id with
 * lgbm_b200_comm_unique_id and hands the bytes to every rank out of band. */
typedef struct lgbm_b200_comm lgbm_b200_comm;
#define LGBM_B200_COMM_ID_BYTES 128
int lgbm_b200_comm_unique_id(uint8_t* id_out);
int lgbm_b200_comm_create(int32_t device, int32_t nranks, int32_t rank, const uint8_t* id,
                          lgbm_b200_comm** out);
int lgbm_b200_comm_destroy(lgbm_b200_comm* comm);

/* Gbdt over this rank's shard. `labels` are the shard's rows in the dataset's
 * order; the global row order is the shards in rank order (the init score is
 * computed from all labels, gathered once). Every rank must call
 * lgbm_b200_booster_train with the same iteration counts. Tree and score
 * accessors work as for lgbm_b200_booster_create; scores are this shard's. */
int lgbm_b200_booster_create_distributed(lgbm_b200_dataset* ds, const float* labels,
                                         const lgbm_b200_train_config* cfg,
                                         lgbm_b200_comm* comm, lgbm_b200_booster** out);

/* ---- Batch prediction from raw feature values (Tree::predict / GetLeaf,
 * lgbm-model/src/tree.rs:193-300; GbdtModel predict, lgbm-model/src/predict.rs) ---- */

/* A tree ensemble: every tree's internal nodes and leaves concatenated, in tree order
 * (borrowed for the create call). Child indices are tree-local: >= 0 an internal node
 * (always greater than its parent's index, as LightGBM numbers nodes), < 0 the leaf ~c.
 * A categorical node's threshold is its index into cat_boundaries over ALL trees;
 * cat_threshold holds the bitsets of real category values (LightGBM model text). */
typedef struct lgbm_b200_model {
  int32_t num_trees;
  int32_t num_features;          /* row width: max_feature_idx + 1 */
  const int32_t* node_offset;    /* [num_trees + 1] */
  const int32_t* leaf_offset;    /* [num_trees + 1] */
  const int32_t* split_feature;  /* [nodes] */
  const double* threshold;       /* [nodes] */
  const int8_t* decision_type;   /* [nodes] bit0 categorical, bit1 default left, bits 2-3 missing type */
  const int32_t* left_child;     /* [nodes] */
  const int32_t* right_child;    /* [nodes] */
  const double* leaf_value;      /* [leaves] */
  int32_t num_cat;
  int32_t transform;             /* 0 identity, 1 sigmoid (binary objective) */
  const int32_t* cat_boundaries; /* [num_cat + 1] */
  const uint32_t* cat_threshold; /* [cat_boundaries[num_cat]] */
  double sigmoid;
} lgbm_b200_model;

typedef struct lgbm_b200_predictor lgbm_b200_predictor;

/* Uploads the ensemble to `device` after checking every index in it. */
int lgbm_b200_predictor_create(int32_t device, const lgbm_b200_model* model,
                               lgbm_b200_predictor** out);
int lgbm_b200_predictor_destroy(lgbm_b200_predictor* p);
/* rows: host row-major f64 [num_rows][num_features]; out: host f64 [num_rows], the sum
 * of the trees' leaf values in tree order, then the model's transform unless raw_score. */
int lgbm_b200_predict(lgbm_b200_predictor* p, const double* rows, int64_t num_rows,
                      int32_t raw_score, double* out);

/* ---- Expert layers: rows routed to experts, products grouped by expert ----
 *
 * The rows of a batch ("tokens") are routed to k of E experts each, the tokens * k slots
 * are grouped by expert, every expert multiplies its ragged range of rows, and a token's
 * k results are joined: learned matrices in ragged ranges of rows, as the leaves of a
 * leaf-wise model are. The calls above do not use them. No counterpart in the reference.
 *
 * Conventions of these entry points
 *  - All array pointers are DEVICE pointers on the current device. The work is enqueued on
 *    `stream` (a cudaStream_t; NULL is the legacy default stream) and not waited for. They
 *    allocate nothing: where scratch is needed the caller passes it, at least as large as
 *    the _workspace function says, 16-byte aligned; it is free again once the stream has
 *    passed the call.
 *  - Pitches are in elements; the innermost axis is contiguous. Outputs are contiguous.
 *    Arrays start at multiples of their elements' size.
 *  - offsets[E + 1], index, chosen and position are device data that the host does not
 *    check. Kernels clamp offsets to the rows given and skip indices outside them.
 *  - At most 512 experts, 16 chosen a token, 2^31 - 65537 rows, products 2^28 wide.
 *  - Sums and softmax statistics are in f32, results rounded once to their type. No result
 *    depends on the order of atomics: the same inputs give the same bits. */
#define LGBM_B200_DTYPE_F32 0
#define LGBM_B200_DTYPE_BF16 1
#define LGBM_B200_DTYPE_F16 2

/* logits [tokens][experts] (pitch >= experts). Per token the k largest logits, ties to the
 * lower expert: chosen (descending logit) and weights, their softmax over the chosen
 * (normalize != 0) or over all experts. -inf is never chosen: a token with fewer than k
 * other logits has chosen -1 and weight 0 in its last slots. NaN ranks first, and its
 * token's weights are NaN. Grouping, stable in slot order: offsets[e] is expert e's first
 * row, offsets[experts] the number of assigned slots; position[slot] is the slot's row (a
 * permutation of tokens * k: slots without an expert come last) and rows[position] its
 * token. */
int64_t lgbm_b200_experts_route_workspace(int64_t tokens, int32_t experts, int32_t k);
int lgbm_b200_experts_route(const void* logits, int32_t dtype, int64_t tokens, int32_t experts,
                            int64_t pitch, int32_t k, int32_t normalize, float* weights,
                            int32_t* chosen, int32_t* position, int32_t* rows, int32_t* offsets,
                            void* workspace, int64_t workspace_bytes, void* stream);
/* dlogits [tokens][experts] of the logits' type from dweights [tokens][k] and the results
 * of lgbm_b200_experts_route on the same logits, k and normalize. */
int lgbm_b200_experts_route_backward(const float* dweights, const float* weights,
                                     const int32_t* chosen, const void* logits, int32_t dtype,
                                     int64_t tokens, int32_t experts, int64_t pitch, int32_t k,
                                     int32_t normalize, void* dlogits, void* stream);

/* Products grouped by expert, bf16 or f16, accumulated in f32; row r belongs to the expert
 * e with offsets[e] <= r < offsets[e + 1]:
 *   y[r]  = w[e] x[index ? index[r] : r]    [rows][outer]; w [experts][outer][inner]
 *   dx[r] = dy[r] w[e]                      [rows][inner]
 *   dw[e] = sum of dy[r]^T x[...]           [experts][outer][inner], of `grad_dtype`: the
 *                                           inputs' type or f32
 * Rows of y and dx that belong to no expert are 0, and so is the dw of an expert without
 * rows. An index outside [0, x_rows) stands for a row of zeros. x, dy and w are read in
 * place when their base and pitch are multiples of 16 bytes, else copied to the workspace
 * first. */
int64_t lgbm_b200_experts_matmul_workspace(const void* x, int64_t x_pitch, const int32_t* index,
                                           const void* w, int64_t rows, int32_t experts,
                                           int32_t inner, int32_t outer);
int lgbm_b200_experts_matmul(const void* x, int64_t x_rows, int64_t x_pitch,
                             const int32_t* index, const void* w, const int32_t* offsets,
                             int32_t dtype, int64_t rows, int32_t experts, int32_t inner,
                             int32_t outer, void* y, void* workspace, int64_t workspace_bytes,
                             void* stream);
/* Both gradients, or one of them: dx or dw NULL is not wanted (w is read for dx only, x for
 * dw only). */
int64_t lgbm_b200_experts_matmul_backward_workspace(const void* dy, int64_t dy_pitch,
                                                    const void* x, int64_t x_pitch,
                                                    const int32_t* index, const void* w,
                                                    int64_t rows, int32_t experts, int32_t inner,
                                                    int32_t outer, int32_t want_dx,
                                                    int32_t want_dw);
int lgbm_b200_experts_matmul_backward(const void* dy, int64_t dy_pitch, const void* x,
                                      int64_t x_rows, int64_t x_pitch, const int32_t* index,
                                      const void* w, const int32_t* offsets, int32_t dtype,
                                      int32_t grad_dtype, int64_t rows, int32_t experts,
                                      int32_t inner, int32_t outer, void* dx, void* dw,
                                      void* workspace, int64_t workspace_bytes, void* stream);
/* Products with what follows them, in the same kernel. act is one of LGBM_B200_ACT_*: relu, silu
 * v / (1 + e^-v), gelu v P(v) with P the distribution function of the normal law.
 *   linear  y[r] = act(w[e] x[..] + bias[e]) + residual[r]     [rows][outer]
 *   gated   h[r] = act(gate) * up                              [rows][hidden], where gate and up
 *           are the first and the last `hidden` columns of w[e] x[..]; w [experts][2 hidden][inner]
 * bias [experts][outer] and residual [rows][outer] (of any pitch) are of the inputs' type; either
 * may be NULL. A row of no expert has y = residual (0 without one) and h = 0.
 * pre (NULL: not wanted) keeps what the activation was given, rounded to the inputs' type, for
 * the backward pass: [rows][ld], gated [rows][2][ld] (gate, then up), ld = the width rounded up
 * to 16, 32-byte aligned; what lies between the width and ld is not defined. Everything before
 * the results' one rounding is in f32. In f16 a value beyond 65504 is saved as an infinity.
 * Workspace: lgbm_b200_experts_linear_workspace with the same operands (gated: outer =
 * 2 hidden). Results overlap none of the inputs. */
#define LGBM_B200_ACT_NONE 0
#define LGBM_B200_ACT_RELU 1
#define LGBM_B200_ACT_SILU 2
#define LGBM_B200_ACT_GELU 3
int64_t lgbm_b200_experts_linear_workspace(const void* x, int64_t x_pitch, const int32_t* index,
                                           const void* w, int64_t rows, int32_t experts,
                                           int32_t inner, int32_t outer);
int lgbm_b200_experts_linear(const void* x, int64_t x_rows, int64_t x_pitch,
                             const int32_t* index, const void* w, const void* bias,
                             const void* residual, int64_t residual_pitch, const int32_t* offsets,
                             int32_t dtype, int32_t act, int64_t rows, int32_t experts,
                             int32_t inner, int32_t outer, void* y, void* pre, void* workspace,
                             int64_t workspace_bytes, void* stream);
int lgbm_b200_experts_gated(const void* x, int64_t x_rows, int64_t x_pitch, const int32_t* index,
                            const void* w, const int32_t* offsets, int32_t dtype, int32_t act,
                            int64_t rows, int32_t experts, int32_t inner, int32_t hidden, void* h,
                            void* pre, void* workspace, int64_t workspace_bytes, void* stream);
/* Their gradients from dy [rows][outer] or dh [rows][hidden] (any pitch) and `pre` as the
 * forward call wrote it (linear without an activation: not read, may be NULL). dx, dw as
 * lgbm_b200_experts_matmul_backward; dbias [experts][outer] of grad_dtype. NULL results are not
 * wanted. The residual's gradient is dy. The gradient of what the activation was given goes to
 * the workspace in the inputs' type, as the matrix products take it: the only rounding between
 * pre and dx, dw, which they hold however wide they are stored. dbias is summed in f32 from its
 * values before that rounding.
 * The range of f16 holds for these steps too, in f32 dw as well: where |dy act'(pre)|, or
 * |dh up act'(gate)| or |dh act(gate)|, passes 65504 the values are infinities, and the row of dx
 * and the row of dw that they enter are not finite; below 2^-25 they are 0. Where pre was saved as
 * an infinity the slopes are their limits, 1 or 0 (relu, silu, gelu), and act(gate) far below zero
 * is 0; act(gate) far above and up are infinite factors. bf16 has f32's range. */
int64_t lgbm_b200_experts_linear_backward_workspace(
    const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, const int32_t* index,
    const void* w, int32_t act, int64_t rows, int32_t experts, int32_t inner, int32_t outer,
    int32_t want_dx, int32_t want_dw, int32_t want_dbias);
int lgbm_b200_experts_linear_backward(const void* dy, int64_t dy_pitch, const void* pre,
                                      const void* x, int64_t x_rows, int64_t x_pitch,
                                      const int32_t* index, const void* w, const int32_t* offsets,
                                      int32_t dtype, int32_t grad_dtype, int32_t act, int64_t rows,
                                      int32_t experts, int32_t inner, int32_t outer, void* dx,
                                      void* dw, void* dbias, void* workspace,
                                      int64_t workspace_bytes, void* stream);
int64_t lgbm_b200_experts_gated_backward_workspace(const void* x, int64_t x_pitch,
                                                   const int32_t* index, const void* w,
                                                   int64_t rows, int32_t experts, int32_t inner,
                                                   int32_t hidden, int32_t want_dx,
                                                   int32_t want_dw);
int lgbm_b200_experts_gated_backward(const void* dh, int64_t dh_pitch, const void* pre,
                                     const void* x, int64_t x_rows, int64_t x_pitch,
                                     const int32_t* index, const void* w, const int32_t* offsets,
                                     int32_t dtype, int32_t grad_dtype, int32_t act, int64_t rows,
                                     int32_t experts, int32_t inner, int32_t hidden, void* dx,
                                     void* dw, void* workspace, int64_t workspace_bytes,
                                     void* stream);
/* y as lgbm_b200_experts_matmul, for a few rows an expert, with weights of 4 bits in groups
 * of group_size (32, 64 or 128) along the inner axis:
 *   w[e][n][k] = scales[e][n][k / group_size] * (q - z)
 * q: the weight's 4 bits, packed like a 4-bit bin row: [experts][outer][stride] bytes, weight
 * 2i in the low half of byte i, stride = ceil(inner / 2) rounded up to 16, 16-byte aligned
 * base. scales: x's type, [experts][outer][ceil(inner / group_size)]. z: zeros[e][n][group]
 * (0..15: its low 4 bits), or 8 where zeros is NULL. Products of q - z are summed in f32 within a group,
 * then scaled in f32: no weight is rounded to 16 bits. */
int lgbm_b200_experts_matmul_w4(const void* x, int64_t x_rows, int64_t x_pitch,
                                const int32_t* index, const uint8_t* q, const void* scales,
                                const uint8_t* zeros, int32_t group_size,
                                const int32_t* offsets, int32_t dtype, int64_t rows,
                                int32_t experts, int32_t inner, int32_t outer, void* y,
                                void* stream);
/* Every wait inside the product kernels is bounded. One that ran out leaves its outputs
 * incomplete and sets a bit here: this call waits for the device, reads the bits of the
 * current device and clears them. */
int lgbm_b200_experts_errors(uint32_t* bits_out);

/* out[t] = sum over j of weights[t][j] * y[position[t][j]] (weights NULL: 1); a position
 * outside [0, rows) adds nothing. */
int lgbm_b200_experts_combine(const void* y, int32_t dtype, int64_t rows, int32_t width,
                              int64_t pitch, const int32_t* position, const float* weights,
                              int64_t tokens, int32_t k, void* out, void* stream);
/* dy[position[t][j]] = weights[t][j] * dout[t]; dweights[t][j] (NULL: not wanted, y is not
 * read) = <dout[t], y[position[t][j]]>. rows must be tokens * k and position a permutation
 * of them, as lgbm_b200_experts_route makes it. */
int lgbm_b200_experts_combine_backward(const void* dout, const void* y, int32_t dtype,
                                       int64_t rows, int32_t width, int64_t dout_pitch,
                                       int64_t pitch, const int32_t* position,
                                       const float* weights, int64_t tokens, int32_t k, void* dy,
                                       float* dweights, void* stream);

/* out = (residual +) x * keep / (1 - p) over rows x width elements numbered row by row.
 * Element i is kept when its 16 random bits are at least D = round(p * 65536); the scale
 * is 65536 / (65536 - D), exact for that D. Bits: Philox4x32-10 of counter (i / 8, offset)
 * and key seed; element i takes the low (i even) or high half of word (i % 8) / 2. The
 * mask is never stored: the gradient of x is the same call on the gradient of out,
 * without a residual. A dropped element is 0 whatever it held. `out` overlaps
 * neither x nor residual. */
int lgbm_b200_experts_dropout(const void* x, const void* residual, int32_t dtype, int64_t rows,
                              int64_t width, int64_t pitch, int64_t residual_pitch, double p,
                              uint64_t seed, uint64_t offset, void* out, void* stream);

/* A step's gradients: *norm (f32, on the device) = sqrt of the sum of the squares of all elements
 * of all tensors, summed so that it is right wherever f32 can hold it. clip_grads also writes
 * out = in * min(1, max_norm / norm): the factor, from the norm as it is returned, is rounded to 24
 * bits (in a wider range than f32's), a product to f32 and then to out's type. In place where out
 * == in (then left alone when the factor is 1), else to other memory that overlaps no tensor read
 * or written. A norm of 0 has the factor 1, and so has any with an infinite max_norm. Where the
 * norm is infinite and max_norm is not, the factor is 0; where the norm is NaN all results are.
 * `tensors` is an array of the HOST, read before the call returns; in and out are contiguous
 * arrays on the current device. The order of the tensors is the order of the sum. */
typedef struct lgbm_b200_experts_tensor {
  const void* in;
  void* out;       /* clip_grads only */
  int64_t count;   /* elements, may be 0 */
  int32_t dtype;   /* LGBM_B200_DTYPE_* */
  int32_t reserved;
} lgbm_b200_experts_tensor;
int64_t lgbm_b200_experts_norm_workspace(const lgbm_b200_experts_tensor* tensors, int64_t count);
int lgbm_b200_experts_grad_norm(const lgbm_b200_experts_tensor* tensors, int64_t count,
                                float* norm, void* workspace, int64_t workspace_bytes,
                                void* stream);
int lgbm_b200_experts_clip_grads(const lgbm_b200_experts_tensor* tensors, int64_t count,
                                 double max_norm, float* norm, void* workspace,
                                 int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LGBM_B200_H */
