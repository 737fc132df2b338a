// The Python side of the 8-bit cache's and the rotary operators, natively: a small call's time is the host's, and reading
// a dozen tensors' shapes, strides and types through Python costs more than the launch.
//
// Each function takes the address of the library entry to call (whichever library _capi routes to), the operator's own
// arguments, checks them, and calls the entry on the current stream of the tensors' device.  A bad argument raises
// ValueError here; a status of the entry itself is returned.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <stdexcept>

#include "morphkv.h"

namespace {

constexpr int64_t kBlock = 16;      // tokens per block
constexpr int64_t kTile = 64;       // tokens the attention kernels take at a time: splits are multiples of it

struct Refused {};                  // a Python error is set

[[noreturn]] void refuse(const char* format, ...) {
    char text[512];
    va_list args;
    va_start(args, format);
    vsnprintf(text, sizeof(text), format, args);
    va_end(args);
    PyErr_SetString(PyExc_ValueError, text);
    throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse("%s must be a tensor", what);
    return THPVariable_Unpack(o);
}

// An attribute of one of the caller's config or state objects.
struct Attr {
    PyObject* value;
    Attr(PyObject* o, PyObject* name) : value(PyObject_GetAttr(o, name)) {
        if (!value) throw Refused{};
    }
    ~Attr() { Py_DECREF(value); }
    Attr(const Attr&) = delete;
    Attr& operator=(const Attr&) = delete;
};

int64_t integer(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        PyObject* as = PyNumber_Index(o);
        if (!as) {
            PyErr_Clear();
            refuse("%s must be an integer", what);
        }
        const long long w = PyLong_AsLongLong(as);
        Py_DECREF(as);
        if (w == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse("%s is out of range", what);
        }
        return w;
    }
    return v;
}

int32_t small(PyObject* o, const char* what) {
    const int64_t v = integer(o, what);
    if (v < INT32_MIN || v > INT32_MAX) refuse("%s is out of range", what);
    return (int32_t)v;
}

struct Names {
    PyObject *num_q_heads, *num_kv_heads, *head_dim, *block_size, *num_prefill_seqs, *num_prefill_tokens, *num_decoding_seqs,
        *max_prefill_len, *max_decoding_len, *softmax_scale, *seq_ids, *prefill_seq_start_locs, *prefill_seq_lens,
        *decoding_seq_lens;
} names;

int32_t int_attr(PyObject* o, PyObject* name) {
    Attr a(o, name);
    return small(a.value, PyUnicode_AsUTF8(name));
}

int32_t dtype_of(const at::Tensor& x, const char* what) {
    const auto t = x.scalar_type();
    if (t != at::kHalf && t != at::kBFloat16) refuse("%s must be float16 or bfloat16", what);
    return t == at::kHalf ? MKV_F16 : MKV_BF16;
}

// Checks x [tokens, heads, dim] against `like`'s type and device; the distance of its rows in elements.
int64_t rows_of(const at::Tensor& x, const char* what, const at::Tensor& like, int64_t tokens, int64_t heads, int64_t dim) {
    if (x.dim() != 3 || x.size(0) != tokens || x.size(1) != heads || x.size(2) != dim)
        refuse("%s must be [%lld, %lld, %lld]", what, (long long)tokens, (long long)heads, (long long)dim);
    if (x.scalar_type() != like.scalar_type() || x.device() != like.device())
        refuse("%s must be of the other rows' type, on their device", what);
    if ((x.stride(2) != 1 && dim != 1) || (x.stride(1) != dim && heads != 1)) refuse("the heads of a row of %s must be contiguous", what);
    return tokens > 1 ? x.stride(0) : heads * dim;
}

// The same for an output, which may also be [tokens, heads * dim]; its rows must not overlap.
int64_t out_rows_of(const at::Tensor& o, const char* what, const at::Tensor& like, int64_t tokens, int64_t heads, int64_t dim) {
    int64_t stride;
    if (o.dim() == 2) {
        if (o.size(0) != tokens || o.size(1) != heads * dim) refuse("%s must be [%lld, %lld]", what, (long long)tokens, (long long)(heads * dim));
        if (o.scalar_type() != like.scalar_type() || o.device() != like.device()) refuse("%s must be of the other rows' type, on their device", what);
        if (o.stride(1) != 1 && heads * dim != 1) refuse("a row of %s must be contiguous", what);
        stride = tokens > 1 ? o.stride(0) : heads * dim;
    } else {
        stride = rows_of(o, what, like, tokens, heads, dim);
    }
    if (stride < heads * dim) refuse("rows of %s overlap", what);
    return stride;
}

// The state's softmax scale.
double scale_of(PyObject* st) {
    const Attr scale(st, names.softmax_scale);
    const double x = PyFloat_AsDouble(scale.value);
    if (x == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("softmax_scale must be a number");
    }
    return x;
}

const int32_t* ints_of(const at::Tensor& t, const char* what, const at::Tensor& like, int64_t least) {
    if (t.scalar_type() != at::kInt || t.device() != like.device() || t.numel() < least || !t.is_contiguous())
        refuse("%s must hold %lld contiguous int32 on the rows' device", what, (long long)least);
    return (const int32_t*)t.const_data_ptr();
}

// The tensors of a state object, kept until the launch is out: one whose attributes are made anew at every access must not
// see its memory handed to the call's own scratch.
struct Held {
    PyObject* objects[8];
    int count = 0;
    Held() = default;
    Held(const Held&) = delete;
    Held& operator=(const Held&) = delete;
    ~Held() {
        while (count > 0) Py_DECREF(objects[--count]);
    }
    const int32_t* ints(PyObject* o, PyObject* name, const at::Tensor& like, int64_t least) {
        PyObject* value = PyObject_GetAttr(o, name);
        if (!value) throw Refused{};
        objects[count++] = value;
        const char* what = PyUnicode_AsUTF8(name);
        return ints_of(tensor(value, what), what, like, least);
    }
};

// Makes the rows' device current for a call, where it is not; its current stream.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const at::Tensor& like) {
        const int here = c10::hip::current_device(), there = like.device().index();
        if (here != there) {
            before = here;
            c10::hip::set_device((c10::DeviceIndex)there);
        }
    }
    ~OnDevice() {
        if (before >= 0) c10::hip::set_device((c10::DeviceIndex)before);
    }
};

void* stream_of(const at::Tensor& like) { return (void*)c10::hip::getCurrentHIPStream(like.device().index()).stream(); }

void on_gpu(const at::Tensor& x, const char* what) {
    if (!x.is_cuda()) refuse("%s must be on the GPU", what);
}

mkv_pool8 pool_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& scales) {
    const auto code = k.scalar_type();
    if ((code != at::kFloat8_e4m3fn && code != at::kChar) || v.scalar_type() != code)
        refuse("an 8-bit cache holds float8_e4m3fn or int8 codes, k and v alike");
    if (k.dim() != 5 || k.numel() == 0) refuse("k must be [num_blocks, L, Hkv, block_size, D], none of them 0");
    const int64_t n = k.size(0), layers = k.size(1), heads = k.size(2), block = k.size(3), dim = k.size(4);
    if (v.dim() != 5 || v.size(0) != n || v.size(1) != layers || v.size(2) != heads || v.size(3) != dim || v.size(4) != block)
        refuse("v must be [num_blocks, L, Hkv, D, block_size] as k's sizes say");
    if (scales.scalar_type() != at::kByte || scales.dim() != 4 || scales.size(0) != layers || scales.size(1) != heads ||
        scales.size(2) != n || scales.size(3) != 2)
        refuse("scales must be uint8 [L, Hkv, num_blocks, 2] as k's sizes say");
    if (!k.is_contiguous() || !v.is_contiguous() || !scales.is_contiguous()) refuse("the tensors of an 8-bit cache must be contiguous");
    if (v.device() != k.device() || scales.device() != k.device()) refuse("the tensors of an 8-bit cache must be on one device");
    if (layers > INT32_MAX || heads > INT32_MAX || block > INT32_MAX || dim > INT32_MAX) refuse("the cache's sizes are out of range");
    mkv_pool8 p = {};
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.scales = (uint8_t*)scales.data_ptr();
    p.num_blocks = n;
    p.num_layers = (int32_t)layers;
    p.num_kv_heads = (int32_t)heads;
    p.block_size = (int32_t)block;
    p.head_dim = (int32_t)dim;
    p.kind = code == at::kChar ? MKV_KV8_INT8 : MKV_KV8_E4M3;
    return p;
}

// The cache, checked against the configs and the rows' device.
mkv_pool8 pool_for(PyObject* const* cache, PyObject* model, PyObject* engine, const at::Tensor& rows) {
    const at::Tensor& k = tensor(cache[0], "cache.k");
    const mkv_pool8 p = pool_of(k, tensor(cache[1], "cache.v"), tensor(cache[2], "cache.scales"));
    if (rows.device() != k.device()) refuse("the rows and the cache are on different devices");
    const int32_t heads = int_attr(model, names.num_kv_heads), dim = int_attr(model, names.head_dim);
    if (p.num_kv_heads != heads || p.head_dim != dim)
        refuse("the cache has %d heads x %d, the model %d x %d", p.num_kv_heads, p.head_dim, heads, dim);
    const int32_t block = int_attr(engine, names.block_size);
    if (p.block_size != block) refuse("the cache has blocks of %d tokens, the engine of %d", p.block_size, block);
    return p;
}

// The step's prefill rows, decode rows or both.
mkv_batch batch_of(const at::Tensor& table, PyObject* st, const at::Tensor& like, bool prefill, bool decode, PyObject* prefix_lens, Held& held) {
    if (table.dim() != 2) refuse("block_table must be [max_seqs, max_blocks_per_seq]");
    mkv_batch b = {};
    b.block_table = ints_of(table, "block_table", like, 0);
    b.table_rows = table.size(0);
    b.max_blocks_per_seq = table.size(1);
    const int32_t seqs = int_attr(st, names.num_prefill_seqs);
    if (seqs < 0) refuse("num_prefill_seqs is negative");
    if (prefill) {
        b.num_prefill_seqs = seqs;
        b.num_prefill_tokens = int_attr(st, names.num_prefill_tokens);
        b.max_prefill_len = int_attr(st, names.max_prefill_len);
    }
    if (decode) b.num_decoding_seqs = int_attr(st, names.num_decoding_seqs);
    const int32_t skipped = prefill ? 0 : seqs;
    b.seq_ids = held.ints(st, names.seq_ids, like, (int64_t)skipped + b.num_prefill_seqs + std::max(b.num_decoding_seqs, 0)) + skipped;
    if (b.num_prefill_seqs) {
        b.prefill_start_locs = held.ints(st, names.prefill_seq_start_locs, like, b.num_prefill_seqs);
        b.prefill_lens = held.ints(st, names.prefill_seq_lens, like, b.num_prefill_seqs);
        if (prefix_lens != Py_None) b.prefix_lens = ints_of(tensor(prefix_lens, "prefix_lens"), "prefix_lens", like, b.num_prefill_seqs);
    }
    if (b.num_decoding_seqs > 0) b.decoding_lens = held.ints(st, names.decoding_seq_lens, like, b.num_decoding_seqs);
    return b;
}

struct Tables {
    const float *cos_t, *sin_t;
    int64_t positions;
    int32_t rotary_dim;
};

Tables tables_of(PyObject* cos_o, PyObject* sin_o, const at::Tensor& like) {
    const at::Tensor &c = tensor(cos_o, "cos"), &s = tensor(sin_o, "sin");
    if (c.dim() != 2 || c.sizes() != s.sizes() || c.scalar_type() != at::kFloat || s.scalar_type() != at::kFloat ||
        !c.is_contiguous() || !s.is_contiguous() || c.device() != like.device() || s.device() != like.device() || c.size(1) > 65535)
        refuse("cos and sin must be contiguous float32 [positions, rotary_dim / 2] on the rows' device");
    return {(const float*)c.const_data_ptr(), (const float*)s.const_data_ptr(), c.size(0), (int32_t)(2 * c.size(1))};
}

int32_t layout_of(PyObject* o) {
    const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (s && !strcmp(s, "half")) return MKV_ROPE_HALF;
    if (s && !strcmp(s, "interleaved")) return MKV_ROPE_INTERLEAVED;
    refuse("layout must be 'half' or 'interleaved'");
}

int compute_units(int device) {
    static int units[64] = {};
    if (device < 0 || device >= 64) return 256;
    if (!units[device]) {
        hipDeviceProp_t prop;
        units[device] = hipGetDeviceProperties(&prop, device) == hipSuccess ? prop.multiProcessorCount : 256;
    }
    return units[device];
}

struct Split {
    int32_t tokens, count;
};

// `splits` ranges, in whole tiles, of `longest` tokens.
Split cut(int64_t longest, int64_t splits) {
    const int64_t tiles = (longest + kTile - 1) / kTile;
    const int64_t per = (tiles + splits - 1) / splits;
    return {(int32_t)(per * kTile), (int32_t)((tiles + per - 1) / per)};
}

// The number of ranges with the least estimated time (`time`, in microseconds, of tiles a range and ranges), of numbers that
// grow by an eighth, up to four rounds of workgroups over `units` compute units.
template <class F>
Split least(int64_t longest, int64_t have, int64_t units, F&& time) {
    longest = std::max<int64_t>(longest, 1);
    const int64_t tiles = (longest + kTile - 1) / kTile;
    const int64_t most = std::min(tiles, std::max<int64_t>(1, 4 * units / have));
    int64_t best = 1;
    double least = 1e300;
    for (int64_t s = 1; s <= most; s += std::max<int64_t>(1, s / 8)) {
        const double t = time((tiles + s - 1) / s, s);
        if (t < least) least = t, best = s;
    }
    return cut(longest, best);
}

// What joining the partials costs: a launch, and 8 bytes written and read for every value at 4.4 TB/s.
double merge_time(int64_t values, int64_t splits) { return splits > 1 ? 3.0 + 1.8e-6 * (double)(values * splits) : 0.0; }

// A decode launch.  A workgroup takes four tiles a step, in 1.5 us where the card has little else to do; a compute unit with
// work from all sides needs 2.3 us (head dim 128) for each of its workgroups' steps, two of them at a time and a third when
// one ends; half a step goes into its beginning and end.  Over 30 batches of random sizes the choice is on average 1.9 %
// slower than the best of sixteen numbers of ranges, where two workgroups per unit, whatever the length, are 8.1 %: 32 rows of
// 1024 to 1536 tokens 17.6 us uncut and 21.1 in two ranges, 12 rows of 3478 with 64 q heads 32.1 us uncut and 23.1 in five.
Split decode_split(int64_t n, int64_t kv_heads, int64_t longest, int64_t units, int64_t q_heads, int64_t dim) {
    const int64_t have = std::max<int64_t>(n * kv_heads, 1);
    units = std::max<int64_t>(units, 1);
    return least(longest, have, units, [&](int64_t tiles, int64_t s) {
        const double load = (double)(have * s) / (double)units;
        const double step = std::max(1.5, 2.3 * (double)dim / 128.0 * (load <= 2.0 ? std::ceil(load) : load + 0.5));
        return ((double)((tiles + 3) / 4) + 0.5) * step + merge_time(n * q_heads * dim, s);
    });
}

// A chunk launch.  A tile of 128 rows takes 1.47 us a key tile where it has a compute unit for itself, and two that share one
// take 1.96; at 64 head dims 1.0, 1.4 for two and 1.9 for three.  Over 30 random batches 1.6 % slower than the best number of
// ranges, where at least four key tiles and two workgroups per unit are 4.1 %: 1024 new tokens 30.4 us uncut and 42.9 in two
// ranges, 128 tokens after 4096 97.5 us uncut, 35.3 in four and 25.7 in eight.
Split prefill_split(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t rows, int64_t keys, int64_t units, int64_t dim) {
    rows = std::max<int64_t>(rows, 1);
    units = std::max<int64_t>(units, 1);
    const int64_t row_tiles = (rows * (q_heads / std::max<int64_t>(kv_heads, 1)) + 127) / 128;
    const int64_t have = std::max<int64_t>(seqs * kv_heads * row_tiles, 1);
    return least(keys, have, units, [&](int64_t tiles, int64_t s) {
        const double load = (double)(have * s) / (double)units;
        const double tile = dim > 64 ? (load <= 1.0 ? 1.47 : 1.96 * std::ceil(load / 2.0))
                                     : (load <= 1.0 ? 1.0 : load <= 2.0 ? 1.4 : 1.9 * std::ceil(load / 3.0));
        return (double)tiles * tile + merge_time(seqs * rows * q_heads * dim, s);
    });
}

Split forced_split(PyObject* o) {
    int tokens, count;
    if (!PyArg_ParseTuple(o, "ii", &tokens, &count)) throw Refused{};
    return {tokens, count};
}

// Partials of a call's output rows and their log sums: torch's allocator hands the memory on in stream order, and a
// captured call gets it from its graph's own pool.
struct Scratch {
    at::Tensor buf;
    float *mid_o = nullptr, *mid_lse = nullptr;
    Scratch(const at::Tensor& like, int64_t rows, int64_t splits, int64_t dim) {
        if (splits <= 1) return;
        buf = at::empty({rows * splits * (dim + 1)}, like.options().dtype(at::kFloat));
        mid_o = (float*)buf.data_ptr();
        mid_lse = mid_o + rows * splits * dim;
    }
};

template <class F>
F* entry(PyObject* o) {
    return (F*)PyLong_AsVoidPtr(o);
}

void expect(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) refuse("%zd arguments, %zd wanted", got, want);
}

// ---- the operators ------------------------------------------------------------------------------------------------------
// (entry, q, k or None, positions, cos, sin, layout, q_out or None, k_out or None)
int rope(PyObject* const* a, Py_ssize_t count) {
    expect(count, 9);
    const at::Tensor& q = tensor(a[1], "q");
    const int32_t dtype = dtype_of(q, "q");
    on_gpu(q, "q");
    if (q.dim() != 3) refuse("q must be [tokens, heads, dim]");
    const int32_t layout = layout_of(a[6]);
    const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
    const at::Tensor& q_out = a[7] == Py_None ? q : tensor(a[7], "q_out");
    const int64_t qs = rows_of(q, "q", q, tokens, heads, dim), qos = out_rows_of(q_out, "q_out", q, tokens, heads, dim);
    const void* k = nullptr;
    void* k_out = nullptr;
    int64_t kv_heads = 0, ks = 0, kos = 0;
    if (a[2] != Py_None) {
        const at::Tensor& kt = tensor(a[2], "k");
        if (kt.dim() != 3) refuse("k must be [tokens, heads, dim]");
        const at::Tensor& ot = a[8] == Py_None ? kt : tensor(a[8], "k_out");
        kv_heads = kt.size(1);
        ks = rows_of(kt, "k", q, tokens, kv_heads, dim);
        kos = out_rows_of(ot, "k_out", q, tokens, kv_heads, dim);
        k = kt.const_data_ptr();
        k_out = ot.data_ptr();
    } else if (a[8] != Py_None) {
        refuse("k_out without k");
    }
    if (heads > INT32_MAX || kv_heads > INT32_MAX || dim > INT32_MAX) refuse("sizes are out of range");
    const at::Tensor& pos = tensor(a[3], "positions");
    if (pos.dim() != 1 || pos.size(0) != tokens) refuse("positions must be [%lld]", (long long)tokens);
    const int32_t* positions = ints_of(pos, "positions", q, tokens);
    const Tables t = tables_of(a[4], a[5], q);
    const OnDevice on(q);
    return entry<decltype(mkv_rope_positions)>(a[0])(dtype, layout, q.const_data_ptr(), k, q_out.data_ptr(), k_out, qs, ks, qos, kos,
                                                     positions, t.cos_t, t.sin_t, t.positions, tokens, (int32_t)heads,
                                                     (int32_t)kv_heads, (int32_t)dim, t.rotary_dim, stream_of(q));
}

// (entry, k, v, cache k, v, scales, block_table, model, engine, state, layer, prefix_lens or None
//  [, q, cos, sin, layout, q_out or None])
int store(PyObject* const* a, Py_ssize_t count) {
    const bool rotates = count == 17;
    if (!rotates) expect(count, 12);
    const at::Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    const int32_t dtype = dtype_of(k, "k");
    on_gpu(k, "k");
    const mkv_pool8 p = pool_for(a + 3, a[7], a[8], k);
    Held held;
    const mkv_batch b = batch_of(tensor(a[6], "block_table"), a[9], k, true, true, a[11], held);
    const int64_t tokens = (int64_t)b.num_prefill_tokens + b.num_decoding_seqs;
    const int64_t ks = rows_of(k, "k", k, tokens, p.num_kv_heads, p.head_dim), vs = rows_of(v, "v", k, tokens, p.num_kv_heads, p.head_dim);
    const int32_t layer = small(a[10], "cur_layer");
    const auto fn = entry<decltype(mkv_store8)>(a[0]);
    if (!rotates) {
        const OnDevice on(k);
        return fn(&p, &b, dtype, k.const_data_ptr(), v.const_data_ptr(), ks, vs, layer, MKV_ROPE_NONE, nullptr, nullptr, 0, 0, 0,
                  nullptr, nullptr, 0, 0, stream_of(k));
    }
    const int32_t heads = int_attr(a[7], names.num_q_heads);
    const int32_t layout = layout_of(a[15]);
    const at::Tensor& q = tensor(a[12], "q");
    const at::Tensor& q_out = a[16] == Py_None ? q : tensor(a[16], "q_out");
    const int64_t qs = rows_of(q, "q", k, tokens, heads, p.head_dim), qos = out_rows_of(q_out, "q_out", k, tokens, heads, p.head_dim);
    const Tables t = tables_of(a[13], a[14], k);
    const OnDevice on(k);
    return fn(&p, &b, dtype, k.const_data_ptr(), v.const_data_ptr(), ks, vs, layer, layout, q.const_data_ptr(), q_out.data_ptr(), qs, qos,
              heads, t.cos_t, t.sin_t, t.positions, t.rotary_dim, stream_of(k));
}

// (entry, q, cache k, v, scales, block_table, model, engine, state, layer, o, split or None)
int decode(PyObject* const* a, Py_ssize_t count) {
    expect(count, 12);
    const at::Tensor &q = tensor(a[1], "q"), &o = tensor(a[10], "o");
    const int32_t dtype = dtype_of(q, "q");
    on_gpu(q, "q");
    const mkv_pool8 p = pool_for(a + 2, a[6], a[7], q);
    Held held;
    const mkv_batch b = batch_of(tensor(a[5], "block_table"), a[8], q, false, true, Py_None, held);
    const int32_t n = b.num_decoding_seqs, heads = int_attr(a[6], names.num_q_heads);
    const int64_t qs = rows_of(q, "q", q, n, heads, p.head_dim), os = out_rows_of(o, "o", q, n, heads, p.head_dim);
    const int32_t layer = small(a[9], "cur_layer");
    if (n == 0) return MKV_OK;
    const double softmax_scale = scale_of(a[8]);
    const int64_t room = b.max_blocks_per_seq * kBlock, known = int_attr(a[8], names.max_decoding_len);
    const OnDevice on(q);
    const Split s = a[11] != Py_None ? forced_split(a[11])
                                     : decode_split(n, p.num_kv_heads, known > 0 ? std::min(known, room) : room, compute_units(q.device().index()),
                                                    heads, p.head_dim);
    const Scratch scratch(q, (int64_t)n * heads, s.count, p.head_dim);
    return entry<decltype(mkv_attn8_decode)>(a[0])(&p, &b, dtype, q.const_data_ptr(), o.data_ptr(), qs, os, heads, (float)softmax_scale,
                                                   layer, s.tokens, s.count, scratch.mid_o, scratch.mid_lse, stream_of(q));
}

// (entry, q, cache k, v, scales, block_table, model, engine, state, layer, o, prefix_lens or None, max_prefix_len, split or None)
int prefill(PyObject* const* a, Py_ssize_t count) {
    expect(count, 14);
    const at::Tensor &q = tensor(a[1], "q"), &o = tensor(a[10], "o");
    const int32_t dtype = dtype_of(q, "q");
    on_gpu(q, "q");
    const mkv_pool8 p = pool_for(a + 2, a[6], a[7], q);
    Held held;
    const mkv_batch b = batch_of(tensor(a[5], "block_table"), a[8], q, true, false, a[11], held);
    const int32_t tokens = b.num_prefill_tokens, heads = int_attr(a[6], names.num_q_heads);
    const int64_t qs = rows_of(q, "q", q, tokens, heads, p.head_dim), os = out_rows_of(o, "o", q, tokens, heads, p.head_dim);
    const int32_t layer = small(a[9], "cur_layer");
    const int64_t max_prefix = integer(a[12], "max_prefix_len");
    if (max_prefix < 0) refuse("max_prefix_len is negative");
    if (b.num_prefill_seqs == 0 || tokens == 0) return MKV_OK;
    const double softmax_scale = scale_of(a[8]);
    const int64_t room = b.max_blocks_per_seq * kBlock;
    const int64_t keys = !b.prefix_lens ? b.max_prefill_len : max_prefix > 0 ? b.max_prefill_len + max_prefix : room;
    const OnDevice on(q);
    const Split s = a[13] != Py_None ? forced_split(a[13])
                                     : prefill_split(b.num_prefill_seqs, heads, p.num_kv_heads, b.max_prefill_len, std::min(keys, room),
                                                     compute_units(q.device().index()), p.head_dim);
    const Scratch scratch(q, (int64_t)tokens * heads, s.count, p.head_dim);
    return entry<decltype(mkv_attn8_prefill)>(a[0])(&p, &b, dtype, q.const_data_ptr(), o.data_ptr(), qs, os, heads, (float)softmax_scale,
                                                    layer, s.tokens, s.count, scratch.mid_o, scratch.mid_lse, stream_of(q));
}

// (q, o, model, state, max_prefix_len): refuses what the attention of a step would, before its append is launched.
int section(PyObject* const* a, Py_ssize_t count) {
    expect(count, 5);
    const at::Tensor &q = tensor(a[0], "q"), &o = tensor(a[1], "o");
    dtype_of(q, "q");
    const int64_t prefill = int_attr(a[3], names.num_prefill_tokens), decode = int_attr(a[3], names.num_decoding_seqs);
    if (prefill < 0 || decode < 0) refuse("num_prefill_tokens or num_decoding_seqs is negative");
    if (decode > 65535) refuse("at most 65535 decode rows per call");
    const int64_t heads = int_attr(a[2], names.num_q_heads), kv_heads = int_attr(a[2], names.num_kv_heads), dim = int_attr(a[2], names.head_dim);
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > 16)
        refuse("num_q_heads %lld must be 1 to 16 times num_kv_heads %lld", (long long)heads, (long long)kv_heads);
    const int64_t qs = rows_of(q, "q", q, prefill + decode, heads, dim), os = out_rows_of(o, "o", q, prefill + decode, heads, dim);
    if ((((uintptr_t)q.const_data_ptr()) & 15) || (qs & 7)) refuse("q rows must be 16-byte aligned");
    if (integer(a[4], "max_prefix_len") < 0) refuse("max_prefix_len is negative");
    const double scale = scale_of(a[3]);
    if (prefill && !(scale > 0)) refuse("softmax_scale must be positive");
    if (prefill && ((((uintptr_t)o.const_data_ptr()) & 15) || (os & 7))) refuse("o rows must be 16-byte aligned");
    return MKV_OK;
}

// No C++ exception leaves a function of the module.
template <class F>
PyObject* guarded(F&& f) noexcept {
    try {
        return f();
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

template <int (*F)(PyObject* const*, Py_ssize_t)>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const int rc = F(args, count);
        return PyErr_Occurred() ? nullptr : PyLong_FromLong(rc);
    });
}

// (k, v, scales) -> the fields of mkv_pool8
PyObject* pool_fields(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        expect(count, 3);
        const mkv_pool8 p = pool_of(tensor(a[0], "k"), tensor(a[1], "v"), tensor(a[2], "scales"));
        return Py_BuildValue("KKKLiiiiii", (unsigned long long)(uintptr_t)p.k, (unsigned long long)(uintptr_t)p.v,
                             (unsigned long long)(uintptr_t)p.scales, (long long)p.num_blocks, p.num_layers, p.num_kv_heads,
                             p.block_size, p.head_dim, p.kind, 0);
    });
}

template <int N>
void numbers(PyObject* const* a, Py_ssize_t count, int64_t (&x)[N]) {
    expect(count, N);
    for (int i = 0; i < N; ++i) x[i] = integer(a[i], "size");
}

PyObject* py_decode_split(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        int64_t x[6];
        numbers(a, count, x);
        const Split s = decode_split(x[0], x[1], x[2], x[3], x[4], x[5]);
        return Py_BuildValue("ii", s.tokens, s.count);
    });
}

PyObject* py_prefill_split(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        int64_t x[7];
        numbers(a, count, x);
        const Split s = prefill_split(x[0], x[1], x[2], x[3], x[4], x[5], x[6]);
        return Py_BuildValue("ii", s.tokens, s.count);
    });
}

PyMethodDef methods[] = {
    {"rope", (PyCFunction)(void (*)(void))call<rope>, METH_FASTCALL, nullptr},
    {"store", (PyCFunction)(void (*)(void))call<store>, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void (*)(void))call<decode>, METH_FASTCALL, nullptr},
    {"prefill", (PyCFunction)(void (*)(void))call<prefill>, METH_FASTCALL, nullptr},
    {"section", (PyCFunction)(void (*)(void))call<section>, METH_FASTCALL, nullptr},
    {"pool_fields", (PyCFunction)(void (*)(void))pool_fields, METH_FASTCALL, nullptr},
    {"decode_split", (PyCFunction)(void (*)(void))py_decode_split, METH_FASTCALL, nullptr},
    {"prefill_split", (PyCFunction)(void (*)(void))py_prefill_split, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
#define MKV_NAME(x)                                         \
    names.x = PyUnicode_InternFromString(#x);               \
    if (!names.x) return nullptr;
    MKV_NAME(num_q_heads)
    MKV_NAME(num_kv_heads)
    MKV_NAME(head_dim)
    MKV_NAME(block_size)
    MKV_NAME(num_prefill_seqs)
    MKV_NAME(num_prefill_tokens)
    MKV_NAME(num_decoding_seqs)
    MKV_NAME(max_prefill_len)
    MKV_NAME(max_decoding_len)
    MKV_NAME(softmax_scale)
    MKV_NAME(seq_ids)
    MKV_NAME(prefill_seq_start_locs)
    MKV_NAME(prefill_seq_lens)
    MKV_NAME(decoding_seq_lens)
#undef MKV_NAME
    return PyModule_Create(&module);
}
