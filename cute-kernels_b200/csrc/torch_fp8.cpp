// The 8-bit operators for torch: argument checks, memory from torch's allocator, autograd nodes, and calls of the C ABI
// (include/fma_b200.h) on the current stream.  They are chains of short launches around small allocations, and a call
// that passes through Python for each of them spends more time there than on the GPU (a training step of a small problem:
// 195 us from Python), so the chains are here; fma_b200/ops/fp8.py holds the documented functions.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "../../include/fma_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

void check(int status, const char* what) {
    TORCH_CHECK(status == FMA_B200_OK, what, " failed: ", fma_b200_status_string(status), " (", fma_b200_last_error(), ")");
}
int32_t dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return FMA_B200_F32;
        case at::kBFloat16: return FMA_B200_BF16;
        case at::kHalf: return FMA_B200_F16;
        default:
            TORCH_CHECK(false, "unsupported dtype ", toString(t), ": the B200 kernels handle float32, bfloat16 and float16");
    }
}
std::string name_of(at::ScalarType t) {  // as Python prints it
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        default: return toString(t);
    }
}
void require_cuda(const Tensor& t) {
    TORCH_CHECK(!t.defined() || t.is_cuda(), "this op runs on CUDA tensors only (no CPU fallback exists)");
}
// There is no forward-mode derivative, and a dual tensor need not require a gradient: without this its tangent would be lost.
void refuse_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name, ": forward-mode derivatives are not available");
}
// The kernels leave no graph behind: a second derivative would come out as none.
void once_differentiable() { TORCH_CHECK(!at::GradMode::is_enabled(), "the 8-bit operators can be differentiated once only (create_graph=False)"); }
void check_cols(const char* name, int64_t cols) {
    TORCH_CHECK(cols >= 8 && cols % 8 == 0, name, ": the width must be a positive multiple of 8, got ", cols);
}
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

int64_t pitch_of(int64_t cols) { return (cols + 15) / 16 * 16; }

// x as [rows, cols] with unit column stride, rows of a single pitch and 16-byte aligned rows; a copy if it has to be.
Tensor rows_2d(const Tensor& x) {
    const int64_t cols = x.size(-1), size = static_cast<int64_t>(x.element_size());
    auto fits = [&](const Tensor& t) {
        return t.dim() == 2 && t.stride(1) == 1 && aligned(t) &&
               (t.size(0) == 1 || (t.stride(0) >= cols && t.stride(0) * size % 16 == 0));
    };
    if (fits(x)) return x;
    // Leading dimensions that collapse onto one pitch are a view, whose derivative is a view too (that of as_strided fills
    // and copies a tensor as large as x's memory).
    const Tensor t = x.reshape({-1, cols});
    return fits(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t pitch_of_rows(const Tensor& x) { return x.size(0) == 1 ? x.size(1) : x.stride(0); }

// 8-bit rows [rows, cols]: one buffer with the values and, behind them, the scales.
struct Held {
    Tensor buffer;
    int64_t rows = 0, cols = 0;
    Held() = default;
    Held(int64_t r, int64_t c, const Tensor& like) : buffer(bytes(r * pitch_of(c) + fma_b200_fp8_scale_bytes(r, c), like)), rows(r), cols(c) {}
    Held(Tensor b, int64_t r, int64_t c) : buffer(std::move(b)), rows(r), cols(c) {}
    uint8_t* values() const { return buffer.data_ptr<uint8_t>(); }
    uint8_t* scales() const { return values() + rows * pitch_of(cols); }
};

Held quantize_rows(const Tensor& x) {
    Held held(x.size(0), x.size(1), x);
    check(fma_b200_fp8_quantize_rows(x.data_ptr(), pitch_of_rows(x), dtype_code(x.scalar_type()), held.rows, held.cols, nullptr,
                                     held.values(), held.scales(), stream_of(x)),
          "fma_b200_fp8_quantize_rows");
    return held;
}
Tensor dequantize(const uint8_t* values, const uint8_t* scales, int64_t batch, int64_t rows, at::IntArrayRef shape, at::ScalarType dtype,
                  const Tensor& like, const int32_t* rows_used) {
    const int32_t code = dtype_code(dtype);
    Tensor out = at::empty(shape, like.options().dtype(dtype));
    if (rows > 0 && batch > 0)
        check(fma_b200_fp8_dequantize(values, scales, static_cast<int32_t>(batch), rows, shape.back(), rows_used, out.data_ptr(), code,
                                      stream_of(like)),
              "fma_b200_fp8_dequantize");
    return out;
}

at::ScalarType scalar_type_or(const py::object& dtype, at::ScalarType otherwise) {
    return dtype.is_none() ? otherwise : torch::python::detail::py_object_to_dtype(dtype);
}

// What quantize_fp8 returns.
struct Blocks {
    Held held;
    std::vector<int64_t> shape;
    at::ScalarType dtype;
    Tensor values() const {
        return held.buffer.narrow(0, 0, held.rows * pitch_of(held.cols)).view(at::kFloat8_e4m3fn).view({held.rows, pitch_of(held.cols)}).narrow(1, 0, held.cols);
    }
    Tensor dequantized(const py::object& to) const {
        require_cuda(held.buffer);
        const c10::cuda::CUDAGuard guard(held.buffer.device());
        return dequantize(held.values(), held.scales(), 1, held.rows, shape, scalar_type_or(to, dtype), held.buffer, nullptr);
    }
};
std::shared_ptr<Blocks> quantize_fp8(const Tensor& x) {
    require_cuda(x);
    dtype_code(x.scalar_type());
    TORCH_CHECK(x.dim() > 0, "quantize_fp8: x needs at least one dimension");
    check_cols("quantize_fp8", x.size(-1));
    const at::NoGradGuard no_grad;
    const c10::cuda::CUDAGuard guard(x.device());
    return std::make_shared<Blocks>(Blocks{quantize_rows(rows_2d(x)), x.sizes().vec(), x.scalar_type()});
}

// What quantize_fp8_weight returns: values, then scales, in one buffer.
struct Weight {
    Tensor buffer;
    std::vector<int64_t> shape;
    at::ScalarType dtype;
    int64_t E, N, K;
    int64_t tiles_rows(int64_t n) const { return E * ((n + 127) / 128) * 128; }
    int64_t value_bytes() const { return E * N * pitch_of(K); }
    int64_t scale_bytes() const { return fma_b200_fp8_scale_bytes(tiles_rows(N), K); }
    uint8_t* values() const { return buffer.data_ptr<uint8_t>(); }
    uint8_t* scales() const { return values() + value_bytes(); }
    Tensor values_tensor() const { return buffer.narrow(0, 0, value_bytes()).view(at::kFloat8_e4m3fn).view({E, N, pitch_of(K)}); }
    Tensor scales_tensor() const { return buffer.narrow(0, value_bytes(), scale_bytes()); }
    Tensor dequantized(const py::object& to) const {
        require_cuda(buffer);
        const c10::cuda::CUDAGuard guard(buffer.device());
        return dequantize(values(), scales(), E, N, shape, scalar_type_or(to, dtype), buffer, nullptr);
    }
};
using WeightPtr = std::shared_ptr<Weight>;

WeightPtr quantize_fp8_weight(const Tensor& weight) {
    require_cuda(weight);
    const int32_t code = dtype_code(weight.scalar_type());
    TORCH_CHECK(weight.dim() == 2 || weight.dim() == 3, "quantize_fp8_weight: weight must be [N, K] or [experts, N, K], got ", weight.sizes());
    check_cols("quantize_fp8_weight", weight.size(-1));
    check_cols("quantize_fp8_weight", weight.size(-2));
    const at::NoGradGuard no_grad;
    const c10::cuda::CUDAGuard guard(weight.device());
    Tensor w = weight.contiguous();
    if (!aligned(w)) w = w.clone();
    auto held = std::make_shared<Weight>(
        Weight{Tensor(), weight.sizes().vec(), weight.scalar_type(), w.dim() == 3 ? w.size(0) : 1, w.size(-2), w.size(-1)});
    held->buffer = bytes(held->value_bytes() + held->scale_bytes(), w);
    check(fma_b200_fp8_quantize_weight(w.data_ptr(), code, static_cast<int32_t>(held->E), static_cast<int32_t>(held->N),
                                       static_cast<int32_t>(held->K), held->values(), held->scales(), stream_of(w)),
          "fma_b200_fp8_quantize_weight");
    return held;
}

// Where rows that are grouped by expert without alignment lie in the 256-aligned layout: one buffer.
struct GroupMaps {
    Tensor buffer;
    int64_t E = 0, layout_rows = 0;
    GroupMaps() = default;
    GroupMaps(Tensor b, int64_t experts, int64_t rows) : buffer(std::move(b)), E(experts), layout_rows(layout_of(experts, rows)) {}
    static int64_t layout_of(int64_t experts, int64_t rows) { return (rows + 255) / 256 * 256 + 256 * std::min(experts, rows); }
    int64_t tiles() const { return layout_rows / 128; }
    int32_t* at(int64_t i) const { return buffer.data_ptr<int32_t>() + i; }
    int32_t* pad_offsets() const { return at(0); }
    int32_t* used() const { return at(E); }          // rows of the layout that experts use
    int32_t* used_all() const { return at(E + 1); }  // and with the rows of no expert
    int32_t* offsets() const { return at(E + 2); }
    int32_t* group_rows() const { return at(2 * E + 3); }
    int32_t* tile_expert() const { return at(3 * E + 3); }
    int32_t* tile_row() const { return at(3 * E + 3 + tiles()); }
    int32_t* tile_rows() const { return at(3 * E + 3 + 2 * tiles()); }
};
int32_t index_bytes(const Tensor& counts) { return counts.scalar_type() == at::kUInt32 ? -4 : static_cast<int32_t>(counts.element_size()); }
GroupMaps make_maps(const Tensor& counts, int64_t rows) {
    const int64_t E = counts.numel();
    GroupMaps m(at::empty({3 * E + 3 + 3 * (GroupMaps::layout_of(E, rows) / 128)}, counts.options().dtype(at::kInt)), E, rows);
    check(fma_b200_fp8_group_maps(counts.data_ptr(), index_bytes(counts), static_cast<int32_t>(E), rows, m.layout_rows,
                                  m.offsets(), m.pad_offsets(), m.group_rows(), m.tile_expert(), m.tile_row(), m.tile_rows(), stream_of(counts)),
          "fma_b200_fp8_group_maps");
    return m;
}
Held quantize_groups(const Tensor& x, const GroupMaps& m, void* copy) {
    Held held(m.layout_rows, x.size(1), x);
    check(fma_b200_fp8_quantize_groups(x.data_ptr(), pitch_of_rows(x), dtype_code(x.scalar_type()), x.size(0), held.cols, m.offsets(),
                                       m.pad_offsets(), static_cast<int32_t>(m.E), m.layout_rows, held.values(), held.scales(), copy,
                                       stream_of(x)),
          "fma_b200_fp8_quantize_groups");
    return held;
}

// [rows, N] = a . w^T, or with `turned` [rows, K] = a . w.
Tensor product(const Held& a, const Weight& w, bool turned, at::ScalarType dtype, int64_t rows, const GroupMaps* m) {
    Tensor out = at::empty({rows, turned ? w.K : w.N}, a.buffer.options().dtype(dtype));
    check((turned ? fma_b200_fp8_gemm_dgrad : fma_b200_fp8_gemm)(
              a.values(), a.scales(), a.rows, w.values(), w.scales(), static_cast<int32_t>(w.E), static_cast<int32_t>(w.N), static_cast<int32_t>(w.K),
              out.data_ptr(), dtype_code(dtype), rows, m ? m->tile_expert() : nullptr, m ? m->tile_row() : nullptr,
              m ? m->tile_rows() : nullptr, m ? m->used_all() : nullptr, nullptr, nullptr, stream_of(out)),
          turned ? "fma_b200_fp8_gemm_dgrad" : "fma_b200_fp8_gemm");
    return out;
}

// Whether the product that reads x itself, in one launch, is the faster way; otherwise x is quantised by a launch of its own
// (with experts also their row maps are made) and the tiles are those of fma_b200_fp8_gemm.  The one launch loses by its CTAs:
// each starts cold, and quantises again the rows that its tile shares with the others of the same rows.  So they are counted: one per
// 128 weight rows and part of the reduction (as few_split deals it, five groups of 512 columns at most; twice where a part is
// longer and an SM has room for one only) for each expert that may be hit, and three for every 16 rows.  The other way costs
// more with experts.  Measured from captured graphs, weights not in L2, this way / the other, us:
//   one matrix  14336 x 4096: 1 row 14.6 / 19.0, 16 rows 18.6 / 19.3, 24 rows 27.3 / 19.4;  28672 x 4096: 8 rows 30.3 / 31.1,
//               16 rows 35.1 / 31.3;  32768 x 8192: 1 row 53.4 / 54.8, 8 rows 58.2 / 55.2;  8192 x 28672: 1 row 73 / 47
//   2 experts   14336 x 4096: 4 rows 28.6 / 38.3, 24 rows 34.6 / 37.7, 48 rows 50.3 / 37.4
//   8 experts   14336 x 4096: 8 rows 59.5 / 63.4, 32 rows 99.3 / 97.6, 128 rows 130 / 98;  4096 x 4096: 64 rows 33.8 / 39.0,
//               128 rows 44.3 / 38.8
//   32 experts  8192 x 4096: 16 rows 84 / 88, 64 rows 183 / 169, 384 rows 246 / 186;  1536 x 2048: 384 rows 28.2 / 33.4
//   128 experts 1536 x 2048: 8 rows 11.5 / 18.9, 512 rows 73 / 89, 1536 rows 91.1 / 90.6;  2048 x 768: 64 rows 24.7 / 30.2, 512 rows
//               58.9 / 52.1;  4096 x 4096: 8 rows 32 / 40, 64 rows 173 / 152
// Over 1276 such cases (1 to 256 experts, 17 shapes, rows spread at random) the faster way is missed by 1.2 % on average.
// Rows that pile up on few experts are not known here; they go 16 at a time all the same.
// In the layer both products go one way, and the other way has more work around them: E = 128, k = 8, H = 2048, I = 768 with 64 /
// 96 / 192 tokens 179 / 190 / 215 against 207 / 209 / 210, E = 8, k = 2, H = 4096, I = 14336 with 4 / 8 / 16 tokens 237 / 288 / 326
// against 254 / 287 / 312.
bool few(int64_t rows, int64_t E, const std::vector<std::pair<int64_t, int64_t>>& shapes) {
    if (rows > 16 * E) return false;
    int64_t ctas = 0;
    for (const auto& [N, K] : shapes) {
        if (K > (1 << 16)) return false;
        const int64_t tiles = (N + 127) / 128, groups = (K + 511) / 512;
        int64_t parts = 1;
        while (parts < 8 && groups > 5 * parts) parts *= 2;
        ctas += tiles * parts * (groups > 5 * parts ? 2 : 1);
    }
    return (16 * std::min(E, rows) + 3 * rows) * ctas <= 16 * (E == 1 ? 1150 : (shapes.size() == 1 ? 3300 : 4000)) * static_cast<int64_t>(shapes.size());
}

Tensor few_rows(const Tensor& x, const Weight& w, const Tensor& counts) {
    Tensor out = at::empty({x.size(0), w.N}, x.options());
    check(fma_b200_fp8_few_rows(x.data_ptr(), pitch_of_rows(x), dtype_code(x.scalar_type()), x.size(0), w.values(), w.scales(),
                                static_cast<int32_t>(w.E), static_cast<int32_t>(w.N), static_cast<int32_t>(w.K),
                                counts.defined() ? counts.data_ptr() : nullptr,
                                counts.defined() ? index_bytes(counts) : 4, out.data_ptr(), stream_of(x)),
          "fma_b200_fp8_few_rows");
    return out;
}

// The 8-bit linear map.  weight: the 16-bit parameter, or none (no gradient of it); counts: rows per expert, or none.
struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const WeightPtr& held,
                          const std::optional<Tensor>& counts, bool want_x, bool want_w) {
        const bool grouped = counts.has_value();
        GroupMaps maps;
        if (grouped) maps = make_maps(*counts, x.size(0));
        const Held rows = grouped ? quantize_groups(x, maps, nullptr) : quantize_rows(x);
        Tensor out = product(rows, *held, false, x.scalar_type(), x.size(0), grouped ? &maps : nullptr);
        ctx->save_for_backward({want_w ? rows.buffer : Tensor(), want_x ? held->buffer : Tensor(), maps.buffer});
        ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), held->E, held->N, held->K, grouped, want_x, want_w};
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable();
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> z = ctx->saved_data["sizes"].toIntVector();
        const int64_t rows = z[0], E = z[1], N = z[2], K = z[3];
        const bool grouped = z[4], want_x = z[5], want_w = z[6];
        const c10::cuda::CUDAGuard guard(grads[0].device());
        const Tensor d_out = rows_2d(grads[0]);
        const at::ScalarType dtype = d_out.scalar_type();
        GroupMaps maps;
        if (grouped) maps = GroupMaps(saved[2], E, rows);
        const int64_t layout = grouped ? maps.layout_rows : rows;
        Tensor d_rows, d_x, d_w;
        Held d8;
        if (!grouped) {
            d_rows = want_w ? d_out.contiguous() : d_out;
            if (want_x) d8 = quantize_rows(d_out);
        } else {
            // the same pass lays the rows out for the weight gradient
            if (want_w) d_rows = at::empty({layout, N}, d_out.options());
            d8 = quantize_groups(d_out, maps, want_w ? d_rows.data_ptr() : nullptr);
        }
        if (want_x) {
            const Weight w{saved[1], {}, dtype, E, N, K};
            d_x = product(d8, w, true, dtype, rows, grouped ? &maps : nullptr);
        }
        if (want_w) {
            const Held x8(saved[0], layout, K);
            const Tensor x_rows = dequantize(x8.values(), x8.scales(), 1, layout, {layout, K}, dtype, d_out, grouped ? maps.used() : nullptr);
            d_w = grouped ? at::empty({E, N, K}, d_out.options()) : at::empty({N, K}, d_out.options());
            check(fma_b200_linear_wgrad(d_rows.data_ptr(), x_rows.data_ptr(), d_w.data_ptr(), dtype_code(dtype), layout, static_cast<int32_t>(E),
                                        static_cast<int32_t>(N), static_cast<int32_t>(K), grouped ? maps.pad_offsets() : nullptr,
                                        grouped ? maps.group_rows() : nullptr, stream_of(d_out)),
                  "fma_b200_linear_wgrad");
        }
        return {d_x, d_w, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear(const char* name, const Tensor& x, const py::object& weight, const Tensor& counts_in, const py::object& quantized) {
    Tensor parameter;
    WeightPtr held;
    if (py::isinstance<Weight>(weight)) {
        held = weight.cast<WeightPtr>();
    } else {
        TORCH_CHECK(THPVariable_Check(weight.ptr()), name, ": weight must be a tensor or what quantize_fp8_weight returns");
        parameter = THPVariable_Unpack(weight.ptr());
        if (!quantized.is_none()) {
            TORCH_CHECK(py::isinstance<Weight>(quantized), name, ": quantized must be what quantize_fp8_weight returns");
            held = quantized.cast<WeightPtr>();
            TORCH_CHECK(parameter.sizes() == held->shape, name, ": quantized has shape ", at::IntArrayRef(held->shape), ", weight ", parameter.sizes());
        }
    }
    Tensor counts = counts_in;
    const at::IntArrayRef shape = parameter.defined() ? parameter.sizes() : at::IntArrayRef(held->shape);
    refuse_tangent(name, x);
    refuse_tangent(name, parameter);
    require_cuda(x);
    require_cuda(parameter);
    require_cuda(counts);
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name, ": x must be bfloat16 or float16, got ", name_of(x.scalar_type()));
    TORCH_CHECK(!parameter.defined() || parameter.scalar_type() == x.scalar_type(), name, ": x is ", name_of(x.scalar_type()), ", weight ",
                name_of(parameter.scalar_type()));
    const bool grouped = counts.defined();
    TORCH_CHECK(shape.size() == (grouped ? 3u : 2u), name, ": unexpected weight shape ", shape);
    const int64_t K = shape.back(), N = shape[shape.size() - 2];
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K, name, ": x ", x.sizes(), " does not fit a weight of shape ", shape);
    if (grouped) {
        TORCH_CHECK(x.dim() == 2, name, ": x must be [rows, ", K, "], got ", x.sizes());
        TORCH_CHECK(counts.dim() == 1 && counts.numel() == shape[0], name, ": expert_frequency must hold one count for each of the ", shape[0], " experts");
        TORCH_CHECK(shape[0] >= 1 && shape[0] <= 1024, name, ": 1 to 1024 experts, got ", shape[0]);
        const at::ScalarType t = counts.scalar_type();
        TORCH_CHECK(t == at::kInt || t == at::kUInt32 || t == at::kLong, name, ": expert_frequency must be int32, uint32 or int64, got ", t);
        TORCH_CHECK(counts.device() == x.device(), name, ": x is on ", x.device(), ", expert_frequency on ", counts.device());
    }
    for (const Tensor& t : {parameter, held ? held->buffer : Tensor()})
        TORCH_CHECK(!t.defined() || t.device() == x.device(), name, ": x is on ", x.device(), ", the weight on ", t.device());
    check_cols(name, N);
    check_cols(name, K);
    const bool grad = at::GradMode::is_enabled();
    const bool want_x = grad && x.requires_grad(), want_w = grad && parameter.defined() && parameter.requires_grad();
    std::vector<int64_t> out_shape = x.sizes().vec();
    out_shape.back() = N;
    const int64_t rows = x.numel() / K;
    if (rows == 0) {
        Tensor out = at::empty(out_shape, x.options());
        // keep the graph: every gradient is zero
        if (want_x) out = out + x.sum() * 0;
        if (want_w) out = out + parameter.sum() * 0;
        return out;
    }
    const c10::cuda::CUDAGuard guard(x.device());
    if (!held) held = quantize_fp8_weight(parameter);
    const Tensor x2 = rows_2d(x);
    if (grouped) counts = counts.contiguous();
    Tensor out;
    if (want_x || want_w) {
        using Maybe = std::optional<Tensor>;
        out = Linear::apply(x2, parameter.defined() ? Maybe(parameter) : Maybe(), held, grouped ? Maybe(counts) : Maybe(), want_x, want_w);
    } else if (few(rows, held->E, {{N, K}})) {
        out = few_rows(x2, *held, counts);
    } else {
        GroupMaps maps;
        if (grouped) maps = make_maps(counts, rows);
        const Held a = grouped ? quantize_groups(x2, maps, nullptr) : quantize_rows(x2);
        out = product(a, *held, false, x.scalar_type(), rows, grouped ? &maps : nullptr);
    }
    return x.dim() == 2 ? out : out.view(out_shape);
}
Tensor linear_fp8(const Tensor& x, const py::object& weight, const py::object& quantized) {
    return linear("linear_fp8", x, weight, Tensor(), quantized);
}
Tensor grouped_linear_fp8(const Tensor& x, const py::object& weight, const Tensor& counts, const py::object& quantized) {
    return linear("grouped_linear_fp8", x, weight, counts, quantized);
}

// SwiGLU; with `kept` also gate and up in 8 bits: a buffer of gate's values, up's values, gate's scales, up's scales.
struct KeptPair {
    int64_t size, scales;
    uint8_t* base;
    KeptPair(const Tensor& buffer, int64_t rows, int64_t cols)
        : size(rows * pitch_of(cols)), scales(fma_b200_fp8_scale_bytes(rows, cols)), base(buffer.data_ptr<uint8_t>()) {}
    uint8_t* gate() const { return base; }
    uint8_t* up() const { return base + size; }
    uint8_t* gate_scales() const { return base + 2 * size; }
    uint8_t* up_scales() const { return base + 2 * size + scales; }
};
Tensor swiglu_forward(const Tensor& gate_in, const Tensor& up_in, Tensor* kept) {
    const Tensor gate = rows_2d(gate_in), up = rows_2d(up_in);
    const int64_t rows = gate.size(0), cols = gate.size(1);
    Tensor out = at::empty(gate_in.sizes(), gate.options());
    if (kept) *kept = bytes(2 * (rows * pitch_of(cols) + fma_b200_fp8_scale_bytes(rows, cols)), gate);
    if (rows == 0) return out;
    uint8_t* at[4] = {nullptr, nullptr, nullptr, nullptr};
    if (kept) {
        const KeptPair k(*kept, rows, cols);
        at[0] = k.gate();
        at[1] = k.gate_scales();
        at[2] = k.up();
        at[3] = k.up_scales();
    }
    check(fma_b200_swiglu_fp8_forward(gate.data_ptr(), pitch_of_rows(gate), up.data_ptr(), pitch_of_rows(up), out.data_ptr(), cols,
                                      dtype_code(gate.scalar_type()), rows, cols, nullptr, at[0], at[1], at[2], at[3], nullptr, nullptr,
                                      stream_of(gate)),
          "fma_b200_swiglu_fp8_forward");
    return out;
}
struct SwigluCheckpoint : torch::autograd::Function<SwigluCheckpoint> {
    static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up) {
        Tensor kept, out = swiglu_forward(gate, up, &kept);
        ctx->save_for_backward({kept});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable();
        const Tensor kept = ctx->get_saved_variables()[0];
        const c10::cuda::CUDAGuard guard(grads[0].device());
        const Tensor d_out = rows_2d(grads[0]);
        const int64_t rows = d_out.size(0), cols = d_out.size(1);
        Tensor gate_grad = at::empty(grads[0].sizes(), d_out.options()), up_grad = at::empty(grads[0].sizes(), d_out.options());
        if (rows > 0) {
            const KeptPair k(kept, rows, cols);
            check(fma_b200_swiglu_fp8_backward(k.gate(), k.gate_scales(), k.up(), k.up_scales(), d_out.data_ptr(), pitch_of_rows(d_out),
                                               gate_grad.data_ptr(), cols, up_grad.data_ptr(), cols, dtype_code(d_out.scalar_type()), rows, cols,
                                               nullptr, nullptr, nullptr, stream_of(d_out)),
                  "fma_b200_swiglu_fp8_backward");
        }
        return {gate_grad, up_grad};
    }
};
Tensor swiglu_fp8_checkpoint(const Tensor& gate, const Tensor& up) {
    TORCH_CHECK(gate.sizes() == up.sizes() && gate.scalar_type() == up.scalar_type() && gate.device() == up.device(),
                "swiglu_fp8_checkpoint: gate and up must have the same shape, dtype and device");
    refuse_tangent("swiglu_fp8_checkpoint", gate);
    refuse_tangent("swiglu_fp8_checkpoint", up);
    require_cuda(gate);
    dtype_code(gate.scalar_type());
    TORCH_CHECK(gate.dim() > 0, "swiglu_fp8_checkpoint: gate needs at least one dimension");
    check_cols("swiglu_fp8_checkpoint", gate.size(-1));
    const c10::cuda::CUDAGuard guard(gate.device());
    if (at::GradMode::is_enabled() && (gate.requires_grad() || up.requires_grad())) return SwigluCheckpoint::apply(gate, up);
    return swiglu_forward(gate, up, nullptr);
}

py::object dtype_object(at::ScalarType t) { return py::reinterpret_borrow<py::object>(reinterpret_cast<PyObject*>(torch::getTHPDtype(t))); }
py::object shape_object(const std::vector<int64_t>& shape) { return py::module_::import("torch").attr("Size")(shape); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::class_<Blocks, std::shared_ptr<Blocks>>(
        m, "Fp8Blocks", "A tensor held in 8 bits, with the shape and dtype it came from: e4m3 values and a scale per 128 columns of a row.")
        .def_property_readonly("values", &Blocks::values, "The e4m3 values without their scales, [rows, cols].")
        .def_property_readonly("nbytes", [](const Blocks& b) { return b.held.buffer.numel(); })
        .def_property_readonly("shape", [](const Blocks& b) { return shape_object(b.shape); })
        .def_property_readonly("dtype", [](const Blocks& b) { return dtype_object(b.dtype); })
        .def_property_readonly("device", [](const Blocks& b) { return py::cast(b.held.buffer).attr("device"); })
        .def("dequantize", &Blocks::dequantized, py::arg("dtype") = py::none(),
             "The values it stands for, rounded to `dtype` (default: the type it was made from).")
        .def(py::pickle(
            [](const Blocks& b) { return py::make_tuple(b.held.buffer, b.held.rows, b.held.cols, b.shape, static_cast<int>(b.dtype)); },
            [](const py::tuple& t) {
                return std::make_shared<Blocks>(Blocks{Held(t[0].cast<Tensor>(), t[1].cast<int64_t>(), t[2].cast<int64_t>()),
                                                       t[3].cast<std::vector<int64_t>>(), static_cast<at::ScalarType>(t[4].cast<int>())});
            }));
    py::class_<Weight, WeightPtr>(m, "Fp8Weight",
                                  "A weight [N, K] or [E, N, K] held in 8 bits with a scale per 128 x 128 block: e4m3 `values` (row pitch: K "
                                  "rounded up to 16) and `scales` in the order in which the tensor cores read them.")
        .def_property_readonly("values", &Weight::values_tensor)
        .def_property_readonly("scales", &Weight::scales_tensor)
        .def_property_readonly("buffer", [](const Weight& w) { return w.buffer; }, "What values and scales lie in.")
        .def_property_readonly(
            "addresses",
            [](const Weight& w) {
                auto at = [](uint8_t* p) { return reinterpret_cast<uintptr_t>(p); };
                return py::make_tuple(at(w.values()), at(w.scales()));
            },
            "Device addresses of values and scales.")
        .def_property_readonly("shape", [](const Weight& w) { return shape_object(w.shape); })
        .def_property_readonly("dtype", [](const Weight& w) { return dtype_object(w.dtype); })
        .def_property_readonly("device", [](const Weight& w) { return py::cast(w.buffer).attr("device"); })
        .def("dequantize", &Weight::dequantized, py::arg("dtype") = py::none(),
             "The values it stands for, rounded to `dtype` (default: the type it was made from).")
        .def(py::pickle(
            [](const Weight& w) { return py::make_tuple(w.buffer, w.shape, static_cast<int>(w.dtype), w.E, w.N, w.K); },
            [](const py::tuple& t) {
                return std::make_shared<Weight>(Weight{t[0].cast<Tensor>(), t[1].cast<std::vector<int64_t>>(),
                                                       static_cast<at::ScalarType>(t[2].cast<int>()), t[3].cast<int64_t>(), t[4].cast<int64_t>(),
                                                       t[5].cast<int64_t>()});
            }));
    for (const char* name : {"Fp8Blocks", "Fp8Weight"}) m.attr(name).attr("__module__") = "fma_b200";  // where pickle finds them
    m.def("few", &few, "Whether this many rows take the one-launch products (rows, experts, [(N, K) of each product]).");
    m.def(
        "refuse_tangents", [](const char* name, const std::vector<Tensor>& tensors) { for (const Tensor& t : tensors) refuse_tangent(name, t); },
        "Raises if one of the tensors carries a forward-mode tangent.");
    m.def("quantize_fp8", &quantize_fp8);
    m.def("quantize_fp8_weight", &quantize_fp8_weight);
    m.def("linear_fp8", &linear_fp8);
    m.def("grouped_linear_fp8", &grouped_linear_fp8);
    m.def("swiglu_fp8_checkpoint", &swiglu_fp8_checkpoint);
}
