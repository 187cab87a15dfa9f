// PyTorch operators of the page tables (gptoss_attn_page_table_update, gptoss_attn_token_map in include/gptoss_attn.h): argument checks, allocation and launch.
#include "torch_direct.h"

namespace {

// The parameter block and the tensors it points into.
struct TableCall {
    gptoss_attn_table_params p{};
    Tensor table, have, want;
};

void fill_lengths(TableCall &c, const Tensor &page_table, const Tensor &have, const Tensor &want, const char *name0, const char *name1, int64_t page_size) {
    TORCH_CHECK(page_table.is_cuda(), "gptoss attention runs on the GPU only (HIP kernels); the page table is on ", page_table.device());
    TORCH_CHECK(page_table.dim() == 2 && is_integers(page_table), "page_table must be (B, pages of a row) integers, got ", page_table.scalar_type(), " ", page_table.sizes());
    for (const auto &[name, t] : {std::pair<const char *, const Tensor &>(name0, have), {name1, want}})
        TORCH_CHECK(t.numel() == page_table.size(0) && is_integers(t), name, " must hold one integer per row, got ", t.scalar_type(), " ", t.sizes(), " for ", page_table.size(0));
    c.have = int32_on(have, page_table).contiguous();
    c.want = int32_on(want, page_table).contiguous();
    gptoss_attn_table_params &p = c.p;
    p.struct_size = sizeof(p);
    p.B = size32(page_table.size(0));
    p.table_width = size32(page_table.size(1));
    TORCH_CHECK(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, "page_size must be a power of two from 16 to 1024, got ", page_size);
    p.page_size = static_cast<int32_t>(page_size);
    p.page_table = const_cast<int32_t *>(c.table.const_data_ptr<int32_t>());
    p.table_stride = p.B == 1 ? 0 : c.table.stride(0);
    p.have = c.have.const_data_ptr<int32_t>();
    p.want = c.want.const_data_ptr<int32_t>();
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Pair page_table_update(const Tensor &page_table, const Tensor &have, const Tensor &want, int64_t pages, int64_t page_size) {
    const c10::OptionalDeviceGuard guard(page_table.device());
    TORCH_CHECK(page_table.scalar_type() == at::kInt && page_table.dim() == 2 && (page_table.stride(1) == 1 || page_table.size(1) <= 1),
                "page_table is written: it must be (B, pages of a row) int32 with contiguous rows, got ", page_table.scalar_type(), " ", page_table.sizes(), " with strides ",
                page_table.strides());
    TableCall c;
    c.table = page_table;
    fill_lengths(c, page_table, have, want, "have", "want", page_size);
    c.p.pages = size32(pages);
    Tensor seqlens = new_tensor({page_table.size(0)}, at::kInt, page_table), left = new_tensor({1}, at::kInt, page_table);
    c.p.seqlens = seqlens.data_ptr<int32_t>();
    c.p.left = left.data_ptr<int32_t>();
    c.p.scratch_bytes = gptoss_attn_table_workspace_bytes(&c.p);
    const Tensor scratch = c.p.scratch_bytes ? new_tensor({static_cast<int64_t>(c.p.scratch_bytes / sizeof(int32_t))}, at::kInt, page_table) : Tensor();
    if (c.p.scratch_bytes) c.p.scratch = scratch.data_ptr();
    about_to_write({&page_table});
    check("gptoss_attn_page_table_update", gptoss_attn_page_table_update(&c.p, stream_of(page_table)));
    return {seqlens, left};
}

using Map = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Map token_map(const Tensor &page_table, const Tensor &start, const Tensor &counts, int64_t total, int64_t page_size) {
    const c10::OptionalDeviceGuard guard(page_table.device());
    TableCall c;
    c.table = page_table;
    if (page_table.dim() == 2 && is_integers(page_table)) {
        c.table = int32_on(page_table, page_table);
        if (c.table.size(1) > 1 && c.table.stride(1) != 1) c.table = c.table.contiguous();
    }
    fill_lengths(c, page_table, start, counts, "start", "counts", page_size);
    TORCH_CHECK(total >= 0 && total <= 1 << 30, "total must be from 0 to 2^30, got ", total);
    gptoss_attn_table_params &p = c.p;
    p.total = static_cast<int32_t>(total);
    Tensor row = new_tensor({total}, at::kInt, page_table), position = new_tensor({total}, at::kInt, page_table), first = new_tensor({total}, at::kInt, page_table);
    Tensor slot = new_tensor({total}, at::kLong, page_table), used = new_tensor({1}, at::kInt, page_table);
    p.used = used.data_ptr<int32_t>();
    // (of no tokens nothing is written)
    p.row = total ? row.data_ptr<int32_t>() : p.used;
    p.position = total ? position.data_ptr<int32_t>() : p.used;
    p.first = total ? first.data_ptr<int32_t>() : p.used;
    p.slot = total ? slot.data_ptr<int64_t>() : reinterpret_cast<int64_t *>(p.used);
    check("gptoss_attn_token_map", gptoss_attn_token_map(&p, stream_of(page_table)));
    return {row, position, slot, first, used};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gptoss_attn, m) {
    m.def("page_table_update(Tensor(a!) page_table, Tensor have, Tensor want, SymInt pages, SymInt page_size) -> (Tensor, Tensor)");
    m.def("token_map(Tensor page_table, Tensor start, Tensor counts, SymInt total, SymInt page_size) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(gptoss_attn, CUDA, m) {
    m.impl("page_table_update", &page_table_update);
    m.impl("token_map", &token_map);
}
#define GPTOSS_TABLES_IMPL(KEY, FN)                                                       \
    TORCH_LIBRARY_IMPL(gptoss_attn, KEY, m) {                                             \
        for (const char *name : {"page_table_update", "token_map"})                       \
            m.impl(name, torch::CppFunction::makeFromBoxedFunction<&FN>());               \
    }
GPTOSS_TABLES_IMPL(Autograd, refuse_gradients)
GPTOSS_TABLES_IMPL(CPU, refuse_cpu)
GPTOSS_TABLES_IMPL(FuncTorchBatched, refuse_vmap)

// Without the dispatcher, as the calls of the cache (torch_paged.cpp).
namespace {

PyObject *update_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &table = a.tensor(0), &have = a.tensor(1), &want = a.tensor(2);
    const int64_t pages = a.integer(3), page_size = a.integer(4);
    if (!a.ok) return not_implemented();
    Pair out;
    {
        const pybind11::gil_scoped_release free;
        out = page_table_update(table, have, want, pages, page_size);
    }
    return pair(out);
    END_HANDLE_TH_ERRORS
}

PyObject *map_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &table = a.tensor(0), &start = a.tensor(1), &counts = a.tensor(2);
    const int64_t total = a.integer(3), page_size = a.integer(4);
    if (!a.ok) return not_implemented();
    Map out;
    {
        const pybind11::gil_scoped_release free;
        out = token_map(table, start, counts, total, page_size);
    }
    pybind11::tuple t(5);
    int i = 0;
    std::apply([&](const auto &...x) { ((t[i++] = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(x))), ...); }, out);
    return t.release().ptr();
    END_HANDLE_TH_ERRORS
}

PyMethodDef kTables[] = {
    {"page_table_update_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&update_now)), METH_FASTCALL, nullptr},
    {"token_map_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&map_now)), METH_FASTCALL, nullptr},
};

}  // namespace

// (page_table_update, token_map) for Python
extern "C" PyObject *gptoss_tables_direct() { return functions_of(kTables); }
