// Compiled operator shim: the per-call path of the four operators that are called once per training
// or Krylov step (SpMV and SpMM, forward and backward) as a torch extension over the C ABI of
// libnumml_b200, in the place of the reference's pybind11 module (cpp/sparse_csr.cpp:300-319, dispatch
// stubs :6-298).  A call does what the reference's ATen glue does -- argument checks, output
// allocation through the caching allocator, current-stream lookup, status to exception -- and nothing
// else: everything that depends on the sparsity pattern only (narrowed index copies, the transposed
// structure, kernel choice, row schedule) is looked up in a small cache keyed on the identity and
// version of the two index tensors.  A cache miss calls back into the Python planner
// (numml_b200/_plan.py), which runs the one-off analysis kernels; the steady state never enters Python
// code beyond the extension call itself.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>

#include <array>
#include <mutex>
#include <vector>

#include "../../include/numml_b200.h"
#include "dense_ops.h"

namespace {

enum Flags { kAutoKernel = 1, kTransposeBackward = 2, kValueSymmetry = 4 };

struct Plan {
    // identity of the pattern
    const void* indices_ptr = nullptr;
    const void* indptr_ptr = nullptr;
    int64_t nnz = 0, rows = 0, cols = 0;
    int device = -1;
    uint32_t indices_version = 0, indptr_version = 0;
    at::Tensor indices_keep, indptr_keep;        // keep the key's addresses from being reused
    // what the kernels read
    at::Tensor idx, ptr;                         // int32 copies, or the int64 originals
    int itype = NB200_I64;
    int block_rows = 0;
    at::Tensor row_order;                        // optional (SpMM, skewed row lengths)
    at::Tensor status;                           // per-device status word
    // transposed structure (built on the first backward)
    bool has_transpose = false;
    at::Tensor t_indptr, t_indices, t_perm, t_row_order;
    int t_block_rows = 0;
    bool pattern_symmetric = false;
    // value symmetry of the last values seen: 0 = seen once, 1 = symmetric, 2 = not symmetric
    const void* values_ptr = nullptr;
    uint32_t values_version = 0;
    int values_state = -1;
    at::Tensor values_keep;
    uint64_t last_use = 0;
};

std::mutex g_mutex;
std::vector<Plan> g_plans;
uint64_t g_clock = 0;
py::object g_resolver;                            // Python: (rows, cols, indices, indptr, transpose) -> dict
constexpr size_t kMaxPlans = 8;

uint32_t version_of(const at::Tensor& t) { return t._version(); }

void check_cuda(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), "numml_b200 operators run on CUDA tensors only (there is no CPU path); ", what, " is on ", t.device());
}

at::Tensor values_tensor(const at::Tensor& t, const at::Tensor* like) {
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kDouble,
                "numml_b200 kernels support float32 and float64, got ", t.scalar_type());
    if (like) TORCH_CHECK(t.scalar_type() == like->scalar_type(), "operands must share one floating type, got ",
                          like->scalar_type(), " and ", t.scalar_type());
    at::Tensor c = t.is_contiguous() ? t : t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
    return c;
}

at::Tensor index_tensor(const at::Tensor& t) {
    TORCH_CHECK(t.scalar_type() == at::kLong, "CSR index arrays must be int64 (as the reference stores them), got ", t.scalar_type());
    return t.is_contiguous() ? t : t.contiguous();
}

int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kDouble ? NB200_F64 : NB200_F32; }

void fill_from(Plan& p, const py::dict& d) {
    p.idx = d["idx"].cast<at::Tensor>();
    p.ptr = d["ptr"].cast<at::Tensor>();
    p.itype = d["itype"].cast<int>();
    p.block_rows = d["block_rows"].cast<int>();
    p.status = d["status"].cast<at::Tensor>();
    if (!d["row_order"].is_none()) p.row_order = d["row_order"].cast<at::Tensor>();
    if (d.contains("t_indptr") && !d["t_indptr"].is_none()) {
        p.t_indptr = d["t_indptr"].cast<at::Tensor>();
        p.t_indices = d["t_indices"].cast<at::Tensor>();
        p.t_perm = d["t_perm"].cast<at::Tensor>();
        p.t_block_rows = d["t_block_rows"].cast<int>();
        p.pattern_symmetric = d["pattern_symmetric"].cast<bool>();
        if (!d["t_row_order"].is_none()) p.t_row_order = d["t_row_order"].cast<at::Tensor>();
        p.has_transpose = true;
    }
}

// The plan of (indices, indptr); `transpose`: the transposed structure is needed too.
Plan& plan_for(int64_t rows, int64_t cols, const at::Tensor& indices, const at::Tensor& indptr, bool transpose) {
    const int device = indices.get_device();
    Plan* found = nullptr;
    for (auto& p : g_plans) {
        if (p.indices_ptr == indices.data_ptr() && p.indptr_ptr == indptr.data_ptr() && p.nnz == indices.numel() &&
            p.rows == rows && p.cols == cols && p.device == device && p.indices_version == version_of(indices) &&
            p.indptr_version == version_of(indptr)) {
            found = &p;
            break;
        }
    }
    if (found && (!transpose || found->has_transpose)) {
        found->last_use = ++g_clock;
        return *found;
    }
    TORCH_CHECK(g_resolver && !g_resolver.is_none(), "numml_b200 extension: no planner registered");
    py::dict d = g_resolver(rows, cols, indices, indptr, transpose).cast<py::dict>();
    if (!found) {
        // drop entries whose key has become stale (same addresses, other version) and the least recently used
        for (size_t q = 0; q < g_plans.size();) {
            if (g_plans[q].indices_ptr == indices.data_ptr() && g_plans[q].indptr_ptr == indptr.data_ptr() && g_plans[q].device == device)
                g_plans.erase(g_plans.begin() + q);
            else
                ++q;
        }
        if (g_plans.size() >= kMaxPlans) {
            size_t lru = 0;
            for (size_t q = 1; q < g_plans.size(); ++q)
                if (g_plans[q].last_use < g_plans[lru].last_use) lru = q;
            g_plans.erase(g_plans.begin() + lru);
        }
        g_plans.emplace_back();
        found = &g_plans.back();
        found->indices_ptr = indices.data_ptr();
        found->indptr_ptr = indptr.data_ptr();
        found->nnz = indices.numel();
        found->rows = rows;
        found->cols = cols;
        found->device = device;
        found->indices_version = version_of(indices);
        found->indptr_version = version_of(indptr);
        found->indices_keep = indices;
        found->indptr_keep = indptr;
    }
    fill_from(*found, d);
    found->last_use = ++g_clock;
    return *found;
}

const void* ptr_or_null(const at::Tensor& t) { return (t.defined() && t.numel() > 0) ? t.data_ptr() : nullptr; }

void check_rc(int rc, const char* fn) { TORCH_CHECK(rc == NB200_OK, fn, " failed: status ", rc, " (", nb200_status_string(rc), ")"); }

// Second sighting of the same values runs the device-side test once; see PatternPlan.values_symmetric.
bool values_symmetric(Plan& p, const at::Tensor& data, cudaStream_t stream) {
    const void* ptr = data.data_ptr();
    const uint32_t ver = version_of(data);
    if (p.values_ptr == ptr && p.values_version == ver && p.values_keep.defined() && p.values_keep.numel() == data.numel()) {
        if (p.values_state == 0) {
            at::Tensor word = at::zeros({1}, data.options().dtype(at::kInt));
            check_rc(nb200_csr_values_symmetric(p.nnz, ptr, p.t_perm.data_ptr(), word.data_ptr<int32_t>(), dtype_code(data),
                                                p.itype, stream), "nb200_csr_values_symmetric");
            p.values_state = word.item<int32_t>() == 0 ? 1 : 2;
        }
        return p.values_state == 1;
    }
    p.values_ptr = ptr;
    p.values_version = ver;
    p.values_state = 0;
    p.values_keep = data;
    return false;
}

at::Tensor spgemv_forward(int64_t rows, int64_t cols, const at::Tensor& A_data, const at::Tensor& A_col_ind,
                          const at::Tensor& A_rowptr, const at::Tensor& x, int flags) {
    check_cuda(A_data, "A_data"); check_cuda(A_col_ind, "A_col_ind"); check_cuda(A_rowptr, "A_rowptr"); check_cuda(x, "x");
    TORCH_CHECK(x.device() == A_data.device() && A_col_ind.device() == A_data.device() && A_rowptr.device() == A_data.device(),
                "all operands must be on the same device");
    const at::Tensor data = values_tensor(A_data, nullptr), xv = values_tensor(x, &data);
    const at::Tensor indices = index_tensor(A_col_ind), indptr = index_tensor(A_rowptr);
    c10::cuda::CUDAGuard guard(data.device());
    std::lock_guard<std::mutex> lock(g_mutex);
    Plan& p = plan_for(rows, cols, indices, indptr, false);
    at::Tensor y = at::empty({rows}, data.options());
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    check_rc(nb200_spgemv_forward(rows, cols, p.nnz, data.data_ptr(), ptr_or_null(p.idx), p.ptr.data_ptr(), nullptr,
                                  ptr_or_null(xv), y.data_ptr(), (flags & kAutoKernel) ? p.block_rows : 0,
                                  p.status.data_ptr<int32_t>(), dtype_code(data), p.itype, stream), "nb200_spgemv_forward");
    return y;
}

std::vector<at::Tensor> spgemv_backward(const at::Tensor& grad_z, int64_t rows, int64_t cols, const at::Tensor& A_data,
                                        const at::Tensor& A_col_ind, const at::Tensor& A_rowptr, const at::Tensor& x, int flags) {
    check_cuda(grad_z, "grad_z"); check_cuda(A_data, "A_data"); check_cuda(A_col_ind, "A_col_ind");
    check_cuda(A_rowptr, "A_rowptr"); check_cuda(x, "x");
    const at::Tensor data = values_tensor(A_data, nullptr), xv = values_tensor(x, &data), g = values_tensor(grad_z, &data);
    const at::Tensor indices = index_tensor(A_col_ind), indptr = index_tensor(A_rowptr);
    c10::cuda::CUDAGuard guard(data.device());
    std::lock_guard<std::mutex> lock(g_mutex);
    const bool transposed = (flags & kTransposeBackward) != 0;
    Plan& p = plan_for(rows, cols, indices, indptr, transposed);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    const bool autok = (flags & kAutoKernel) != 0;
    const int block_rows = autok ? p.block_rows : 0;
    const int t_block_rows = (autok && transposed) ? p.t_block_rows : 0;
    int symmetry = (autok && transposed && block_rows > 0 && p.pattern_symmetric) ? NB200_SYMMETRIC_PATTERN : 0;
    if (symmetry && (flags & kValueSymmetry) && values_symmetric(p, data, stream)) symmetry |= NB200_SYMMETRIC_VALUES;
    at::Tensor grad_A = at::empty_like(data);
    at::Tensor grad_x = at::empty({cols}, data.options());
    check_rc(nb200_spgemv_backward(rows, cols, p.nnz, data.data_ptr(), ptr_or_null(p.idx), p.ptr.data_ptr(), ptr_or_null(xv),
                                   ptr_or_null(g), transposed ? p.t_indptr.data_ptr() : nullptr,
                                   transposed ? ptr_or_null(p.t_indices) : nullptr, transposed ? ptr_or_null(p.t_perm) : nullptr,
                                   grad_A.data_ptr(), grad_x.data_ptr(), block_rows, t_block_rows, symmetry,
                                   p.status.data_ptr<int32_t>(), dtype_code(data), p.itype, stream), "nb200_spgemv_backward");
    return {grad_A, grad_x};
}

at::Tensor spdmm_forward(int64_t rows, int64_t cols, const at::Tensor& A_data, const at::Tensor& A_indices,
                         const at::Tensor& A_indptr, const at::Tensor& B) {
    check_cuda(A_data, "A_data"); check_cuda(A_indices, "A_indices"); check_cuda(A_indptr, "A_indptr"); check_cuda(B, "B");
    TORCH_CHECK(B.dim() == 2, "expected a 2-D dense matrix, got ", B.dim(), " dimensions");
    TORCH_CHECK(B.size(0) == cols, "dense operand has ", B.size(0), " rows, expected ", cols);
    const at::Tensor data = values_tensor(A_data, nullptr), Bv = values_tensor(B, &data);
    const at::Tensor indices = index_tensor(A_indices), indptr = index_tensor(A_indptr);
    c10::cuda::CUDAGuard guard(data.device());
    std::lock_guard<std::mutex> lock(g_mutex);
    Plan& p = plan_for(rows, cols, indices, indptr, false);
    const int64_t K = Bv.size(1);
    at::Tensor C = at::empty({rows, K}, data.options());
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    check_rc(nb200_spdmm_forward(rows, cols, K, p.nnz, data.data_ptr(), ptr_or_null(p.idx), p.ptr.data_ptr(), nullptr,
                                 static_cast<const int32_t*>(ptr_or_null(p.row_order)), ptr_or_null(Bv), C.data_ptr(),
                                 dtype_code(data), p.itype, stream), "nb200_spdmm_forward");
    return C;
}

std::vector<at::Tensor> spdmm_backward(int64_t rows, int64_t cols, const at::Tensor& A_data, const at::Tensor& A_indices,
                                       const at::Tensor& A_indptr, const at::Tensor& B, const at::Tensor& grad_C) {
    check_cuda(A_data, "A_data"); check_cuda(A_indices, "A_indices"); check_cuda(A_indptr, "A_indptr");
    check_cuda(B, "B"); check_cuda(grad_C, "grad_C");
    TORCH_CHECK(B.dim() == 2 && grad_C.dim() == 2, "expected 2-D dense matrices");
    const at::Tensor data = values_tensor(A_data, nullptr), Bv = values_tensor(B, &data), G = values_tensor(grad_C, &data);
    const at::Tensor indices = index_tensor(A_indices), indptr = index_tensor(A_indptr);
    c10::cuda::CUDAGuard guard(data.device());
    std::lock_guard<std::mutex> lock(g_mutex);
    Plan& p = plan_for(rows, cols, indices, indptr, true);
    const int64_t K = Bv.size(1);
    at::Tensor grad_A = at::empty_like(data);
    at::Tensor grad_B = at::empty({cols, K}, data.options());
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    const int code = dtype_code(data);
    check_rc(nb200_spdmm_backward_grad_A(rows, cols, K, p.nnz, ptr_or_null(p.idx), p.ptr.data_ptr(),
                                         static_cast<const int32_t*>(ptr_or_null(p.row_order)), ptr_or_null(Bv), ptr_or_null(G),
                                         grad_A.data_ptr(), code, p.itype, stream), "nb200_spdmm_backward_grad_A");
    // grad_B = A^T grad_C: the forward kernel over the transposed structure, values through the permutation
    check_rc(nb200_spdmm_forward(cols, rows, K, p.nnz, data.data_ptr(), ptr_or_null(p.t_indices), p.t_indptr.data_ptr(),
                                 ptr_or_null(p.t_perm), static_cast<const int32_t*>(ptr_or_null(p.t_row_order)), ptr_or_null(G),
                                 grad_B.data_ptr(), code, p.itype, stream), "nb200_spdmm_forward");
    return {grad_A, grad_B};
}

void set_planner(py::object resolver) {
    std::lock_guard<std::mutex> lock(g_mutex);
    g_resolver = std::move(resolver);
}

void clear_plans() {
    std::lock_guard<std::mutex> lock(g_mutex);
    g_plans.clear();
}

// Last state of the value-symmetry test of a pattern, for the tests: -1 unknown, 0 seen once, 1 yes, 2 no.
int values_state(const at::Tensor& indices, const at::Tensor& indptr) {
    std::lock_guard<std::mutex> lock(g_mutex);
    for (auto& p : g_plans)
        if (p.indices_ptr == indices.data_ptr() && p.indptr_ptr == indptr.data_ptr()) return p.values_state;
    return -1;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "compiled per-call path of numml_b200's SpMV / SpMM operators and dense operators over libnumml_b200";
    register_dense_ops(m);
    m.def("spgemv_forward", &spgemv_forward);
    m.def("spgemv_backward", &spgemv_backward);
    m.def("spdmm_forward", &spdmm_forward);
    m.def("spdmm_backward", &spdmm_backward);
    m.def("set_planner", &set_planner);
    m.def("clear_plans", &clear_plans);
    m.def("values_state", &values_state);
    m.def("library_version", []() { return nb200_version(); });
    // the planner and the cached tensors are released while the interpreter is still alive
    py::module_::import("atexit").attr("register")(py::cpp_function([]() {
        std::lock_guard<std::mutex> lock(g_mutex);
        g_plans.clear();
        g_resolver = py::object();
    }));
}
