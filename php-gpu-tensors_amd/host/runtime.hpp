// Host runtime of the MI355X backend: the C++ counterpart of the reference's
// tensor runtime and op dispatch (src/tensor.c, src/operations.c,
// src/cuda_array/ca_private.c, the cuda_array_ce.c composites and the Fusion
// compiler src/fusion_*.c).  It owns tensor metadata, applies the
// reference's dtype/shape rules, and reaches the GPU only through the C-ABI
// of include/pt_hip.h.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <memory>
#include <string>
#include <vector>

#include "../../include/pt_hip.h"

namespace phpt {

constexpr int kMaxDims = 10;        // MAX_DIMS, src/tensor.h:16
constexpr int kGlobalAxis = -1000;  // REDUCE_GLOBAL_FLAG analogue

// ------------------------------------------------------------------ errors
enum ErrorKind { ERR_NONE = 0, ERR_INVALID = 1, ERR_RUNTIME = 2 };
void set_invalid(const char *fmt, ...);
void set_runtime(const char *fmt, ...);
void clear_error();
int error_kind();
const char *error_message();
bool check_status(pt_status st, const char *what);  // false + error set on failure
pt_status last_failed_status();  // status of the latest check_status that failed
void reset_failed_status();

// ------------------------------------------------------------------ dtypes
// dtype_t numbering of src/data_types.h:8-25 (PT_* codes).
size_t dtype_size(int dt);
bool is_floating(int dt);
bool is_integer(int dt);
bool is_signed(int dt);
bool is_valid_dtype(int dt);
const char *dtype_name(int dt);
int dtype_from_name(const char *name);

// Scalar value with its dtype, as scalar_value_t (src/data_types.h:38-59).
struct Scalar {
    int dtype = PT_FLOAT64;
    double f = 0.0;       // float32/float64/float16/bfloat16 value (as double)
    int64_t i = 0;        // signed integers
    uint64_t u = 0;       // unsigned integers / bool
    bool is_neg = false;
    long double as_ld() const;
};
Scalar scalar_from_double(double v);
Scalar scalar_from_int(int64_t v);
Scalar scalar_from_bool(bool v);
// cast_single_value (data_types.c:373-436); returns false when the value is
// not representable (integer range), leaving `out` unchanged.
bool cast_scalar(const Scalar &in, int target, Scalar &out);
pt_scalar_t to_pt_scalar(const Scalar &s);

int promote_types(int a, int b);                                // :301-349
int promote_scalar_for_arithmetic(int t, int s, int op, bool is_neg);  // :438-490
int promote_types_for_arithmetic(int a, int b, int op);        // :492-516
bool can_safely_cast_to(int from, int to);                      // :570-629

// ------------------------------------------------------------------ tensors
struct Storage {
    void *ptr = nullptr;
    size_t bytes = 0;
    Storage() = default;
    Storage(const Storage &) = delete;
    Storage &operator=(const Storage &) = delete;
    ~Storage();
};

struct FusionNode;

struct Tensor {
    std::shared_ptr<Storage> storage;
    int dtype = PT_FLOAT32;
    int ndims = 0;
    int shape[kMaxDims] = {0};
    size_t strides[kMaxDims] = {0};  // elements
    size_t offset = 0;               // elements
    bool read_only = false;          // broadcast views
    bool is_view = false;            // made by a view operation (shares storage)
    bool fusion_failed = false;      // recorded in a Fusion scope that was aborted
    std::shared_ptr<FusionNode> node;  // set while recorded in a Fusion scope
    uint64_t id = 0;

    size_t numel() const;
    bool contiguous() const;
    bool lazy() const { return node != nullptr && !storage; }
    void *data() const;
    std::vector<int> shape_vec() const { return std::vector<int>(shape, shape + ndims); }
};
using TensorP = std::shared_ptr<Tensor>;

uint64_t next_tensor_id();
void contiguous_strides(const int *shape, int ndims, size_t *strides);
bool shape_metrics(const int *shape, int ndims, size_t *elements);  // tensor_shape_metrics
bool broadcast_shape(const int *a, int na, const int *b, int nb, int *out, int *nout);
bool matmul_shape(const int *a, int na, const int *b, int nb, int *out, int *nout);

TensorP make_empty(const int *shape, int ndims, int dtype);  // allocated, uninitialised
TensorP make_meta(const int *shape, int ndims, int dtype);   // metadata only (lazy)
// bytes of a contiguous tensor; SIZE_MAX, which no allocation serves, where they overflow
size_t storage_bytes(const Tensor &t);
TensorP from_host(const void *data, const int *shape, int ndims, int dtype);
bool to_host(const TensorP &t, void *out, size_t bytes);     // logical row-major bytes
TensorP full(const int *shape, int ndims, int dtype, const Scalar &value);
TensorP materialize(const TensorP &t);                       // contiguous copy if needed

// Native steps of a plan captured into a HIP graph must not allocate: while
// allocation_forbidden() is set, make_empty fails.  A plan hands a native
// step its (stable) output buffer with preset_output; the native operation
// takes it through output_tensor when shape and dtype match.
bool &allocation_forbidden();
uint64_t allocation_refusals();  // allocations refused while forbidden (this thread)
void preset_output(const TensorP &t);
TensorP output_tensor(const int *shape, int ndims, int dtype);

// views (share storage)
TensorP view(const TensorP &t, const int *shape, const size_t *strides, int ndims, size_t offset);
TensorP reshape(const TensorP &t, const int *shape, int ndims);
TensorP transpose(const TensorP &t, const int *perm, int nperm);
TensorP broadcast_to(const TensorP &t, const int *shape, int ndims);
TensorP slice_axis(const TensorP &t, int axis, int start, int stop, int step);
TensorP select_index(const TensorP &t, int axis, int index);

// ------------------------------------------------------------------ eager ops
// Names and validation follow src/cuda_array/ca_private.c.
TensorP cuda_tensor_op(const TensorP &a, const TensorP &b, int op);
TensorP cuda_scalar_op(const TensorP &a, const Scalar &s, int op);
TensorP cuda_inv_scalar_op(const TensorP &a, const Scalar &s, int op);
TensorP cuda_unary_op(const TensorP &a, int op);
TensorP cuda_tensor_reduce(const TensorP &a, int axis, int op);      // axis may be kGlobalAxis
TensorP cuda_tensor_reduce_arg(const TensorP &a, int axis, int op);  // axis may be kGlobalAxis
TensorP cuda_array_variance(const TensorP &a, int axis, long correction, bool std_dev);
TensorP cuda_array_softmax(const TensorP &a, int axis);
TensorP cuda_array_layernorm(const TensorP &a, const int *axes, int naxes, double eps,
                             const TensorP &scale, const TensorP &bias);
TensorP cuda_tensor_matmul(const TensorP &a, const TensorP &b);
TensorP cuda_tune_matmul(const TensorP &a, const TensorP &b, int *tiles, float *median_ms, int max_candidates,
                         int *count, int *selected);
TensorP cuda_tensor_where(const TensorP &c, const TensorP &x, const TensorP &y);
// gather / scatterAdd along `axis` (ca_private.c:916-1007); int32 indices
TensorP cuda_tensor_gather(const TensorP &input, const TensorP &indices, int axis);
TensorP cuda_tensor_scatter_add(const TensorP &input, const TensorP &indices, const TensorP &updates, int axis);
// validation record of the executing Fusion plan (nullptr outside one)
int32_t *&index_record();
// Where the sequences of a packed tensor, or of the slots of a cache, lie
// among its token rows.  Checked on the host when it is made and never
// changed; the device copy is int32 [2, count], starts then lengths.
struct Sequences {
    std::vector<int> starts, lengths;
    int most = 0;          // longest
    long long end = 0;     // first row past the last sequence
    long long total = 0;   // rows of all sequences
    bool overlap = false;  // some row lies in two of them
    TensorP device;
    int count() const { return (int)lengths.size(); }
    const int32_t *device_starts() const;
    const int32_t *device_lengths() const;
    // every row of a tensor of `rows` lies in one sequence
    bool cover(long long rows) const { return !overlap && total == rows; }
};
using SequencesP = std::shared_ptr<Sequences>;
SequencesP make_sequences(const int *lengths, const int *starts, int count);  // starts null: one behind the other

// Operators with several results: `out` gets one tensor per result (null
// where it is not wanted).  lse and, for 16-bit operands, rest are kept for
// the gradient.
bool cuda_array_attention(const TensorP &q, const TensorP &k, const TensorP &v, bool causal, double scale,
                          const SequencesP &qs, const SequencesP &ks, bool keep, TensorP out[3]);
bool cuda_array_attention_backward(const TensorP &q, const TensorP &k, const TensorP &v, const TensorP &o,
                                   const TensorP &lse, const TensorP &rest, const TensorP &grad, bool causal,
                                   double scale, const SequencesP &qs, const SequencesP &ks, TensorP out[3]);
// layerNorm's checks; axes (at most kMaxDims) without negative ones
bool layernorm_axes(const TensorP &a, const int *axes_in, int naxes, double eps, const TensorP &scale, const TensorP &bias,
                    int *axes);
// gradients of the input, the scale and the bias; scale and bias may be null
bool cuda_array_layernorm_backward(const TensorP &a, const TensorP &grad, const int *axes, int naxes, double eps,
                                   const TensorP &scale, const TensorP &bias, TensorP out[3]);
// log probability, entropy, stats [.., 2], log probabilities and indices of the `top` likeliest
bool cuda_array_logprobs(const TensorP &a, const TensorP &tokens, int top, TensorP out[5]);
TensorP cuda_array_logprobs_backward(const TensorP &a, const TensorP &tokens, const TensorP &stats, const TensorP &entropy,
                                     const TensorP &top_index, const TensorP &g_logprob, const TensorP &g_entropy,
                                     const TensorP &g_top);
// Frequencies of a rotation by position: part / 2 of them on the device, in
// turns a position.  Checked when it is made and never changed.
struct Rotary {
    int part = 0;
    bool interleaved = false;
    double magnitude = 1.0;
    TensorP turns;
};
using RotaryP = std::shared_ptr<Rotary>;
RotaryP make_rotary(int part, double base, bool interleaved, double factor, double context, double low, double high,
                    double magnitude, const double *frequencies);
// k, positions, qs and ks may be null; out: the turned q and, with k, k
bool cuda_array_rotary(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan, const TensorP &qs,
                       const TensorP &ks, double eps, TensorP out[2]);
// gq or gk null: that side has no gradient; out: of q, k, qs, ks
bool cuda_array_rotary_backward(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan,
                                const TensorP &qs, const TensorP &ks, double eps, const TensorP &gq, const TensorP &gk,
                                TensorP out[4]);
// act(x gate) * (x up) over the last axis of x; out: the result and, with
// keep, both products for the gradient: uint8 [bytes, rows, columns]
bool cuda_array_gated(const TensorP &x, const TensorP &gate, const TensorP &up, int activation, bool keep, TensorP out[2]);
// out: of x, gate and up (null where not wanted)
bool cuda_array_gated_backward(const TensorP &x, const TensorP &gate, const TensorP &up, const TensorP &kept,
                               const TensorP &grad, int activation, bool want_x, bool want_weights, TensorP out[3]);
// One AdamW step over many tensors; the state's arrays in the order
// first, second, power1, power2, then with masters master, then with 8-bit
// moments first's and second's exponents and draws.
struct AdamwStep {
    int bits = 32;
    bool master = false, has_rate = false;
    double beta1 = 0, beta2 = 0, epsilon = 0, weight_decay = 0, rate = 0;
    std::vector<uint8_t> decay;
    int count() const { return (int)decay.size(); }
    int states() const { return 4 + master + (bits == 8 ? 3 : 0); }
};
using AdamwStepP = std::shared_ptr<const AdamwStep>;
// out: the parameters, then the states
bool cuda_array_adamw(const AdamwStepP &step, const std::vector<TensorP> &params, const std::vector<TensorP> &grads,
                      const std::vector<TensorP> &states, const TensorP &rate, std::vector<TensorP> &out);
long long adamw_blocks(const std::vector<TensorP> &params);  // -1: too many
TensorP cuda_array_adamw_masters(const std::vector<TensorP> &params);
bool cuda_array_adamw_moments(const TensorP &first, const TensorP &first_exponent, const TensorP &second,
                              const TensorP &second_exponent, TensorP out[2]);
TensorP tensor_cast(const TensorP &a, int dtype);
TensorP astype(const TensorP &a, int dtype);  // safe casts only (CudaArray::astype)
TensorP copy(const TensorP &a);

// ------------------------------------------------------------------ fusion
// Recording mirrors src/fusion_capture.c: inside a Fusion scope every op on
// CudaArray values appends a node and returns a lazy tensor (shape and
// dtype known, no storage).
enum NodeKind {
    N_INPUT = 0,   // placeholder bound at run time (Fusion::compile inputs)
    N_BINARY,      // tensor (op) tensor
    N_SCALAR,      // tensor (op) scalar, or scalar (op) tensor when reverse
    N_UNARY,
    N_CAST,
    N_WHERE,
    N_VIEW,        // affine index map over the source's logical layout
    N_NATIVE       // boundary op executed by a native kernel
};

enum NativeKind {
    NAT_MATMUL = 0, NAT_REDUCE, NAT_ARG_REDUCE, NAT_MOMENTS, NAT_SOFTMAX, NAT_LAYERNORM, NAT_GATHER, NAT_SCATTER_ADD,
    // A native step has one result.  Further results of an operator are
    // buffers that the step gets as operands and writes: NAT_BUFFER makes one
    // (no kernel), and NAT_RESULT is its value once the step in its second
    // operand has written it.
    NAT_BUFFER, NAT_RESULT,
    NAT_ATTENTION, NAT_ATTENTION_BACKWARD, NAT_LAYERNORM_BACKWARD, NAT_LOGPROBS, NAT_LOGPROBS_BACKWARD,
    NAT_ROTARY, NAT_ROTARY_BACKWARD, NAT_GATED, NAT_GATED_BACKWARD, NAT_ADAMW, NAT_ADAMW_MOMENTS
};

struct NativeSpec {
    int kind = NAT_MATMUL;
    int op = 0;
    int axis = 0;
    long correction = 0;
    bool std_dev = false;
    double eps = 0.0;
    int naxes = 0;
    int axes[kMaxDims] = {0};
    bool has_scale = false, has_bias = false;
    bool causal = false;
    int activation = 0;
    int top = 0, given = 0;  // given: which optional operands follow (a bit each)
    SequencesP q_seq, k_seq;
    RotaryP rotary;
    AdamwStepP adamw;
};

struct FusionNode {
    NodeKind kind = N_INPUT;
    int op = 0;
    std::vector<TensorP> inputs;
    Scalar scalar;
    bool reverse = false;
    // N_VIEW: out index -> source linear index = offset + sum coord_d * stride_d
    size_t view_strides[kMaxDims] = {0};
    size_t view_offset = 0;
    NativeSpec native;
    int input_index = -1;  // N_INPUT: position in the compile() input list
};

bool fusion_active();
TensorP fusion_record(NodeKind kind, int op, std::vector<TensorP> inputs, const int *shape,
                      int ndims, int dtype);
TensorP fusion_record_scalar(const TensorP &a, const Scalar &s, int op, bool reverse, int dtype);
TensorP fusion_record_view(const TensorP &a, const int *shape, const size_t *strides, int ndims,
                           size_t offset);
TensorP fusion_record_native(const NativeSpec &spec, std::vector<TensorP> inputs, const int *shape,
                             int ndims, int dtype);
// Execute the recorded graph that produces a lazy tensor (in-scope
// materialization, e.g. toArray() inside Fusion::run) and attach storage.
bool fusion_materialize(const TensorP &t);

// Eager implementations of native boundary ops (inputs materialized).
TensorP native_execute(const NativeSpec &spec, const std::vector<TensorP> &inputs);
TensorP native_execute_model(const NativeSpec &spec, const std::vector<TensorP> &inputs);  // model_ops.cpp
TensorP native_execute_block(const NativeSpec &spec, const std::vector<TensorP> &inputs);  // block_ops.cpp
// A further result of the native step `main` (see NativeKind), its buffer
// recorded before the step.
TensorP record_buffer(const int *shape, int nd, int dtype);
TensorP record_result(const TensorP &buffer, const TensorP &main);
bool low_or_f32(int dt);
bool same_shape(const Tensor &a, const Tensor &b);
// A tensor whose last axis is read with its elements side by side: itself
// where they lie so, else packed.  strides (of rank 3 or 4): sequence, token, head.
TensorP head_operand(const TensorP &t, size_t strides[3]);
bool guard(const TensorP &t);  // materialized, or an error set
}  // namespace phpt

// Opaque C handles of phpt_host.h: one reference each.
struct phpt_tensor {
    phpt::TensorP t;
};
struct phpt_sequences {
    phpt::SequencesP s;
};
struct phpt_rotary_plan {
    phpt::RotaryP p;
};
