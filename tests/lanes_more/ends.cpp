// Parts of the page kernels over a row's last columns alone, at widths that no test on
// the CPU could go through from the start.
#include "qwen2_pages.hip"

namespace w4g64 {
namespace {

struct EndsArgs {
    ResizeArgs a;
    uint32_t from;
    int free, length;
    int32_t* said;  // entries that lack a page, and what name one afterwards
};

void ends_kernel(EndsArgs e) {
    Columns first;
    first.load(e.a.table, e.from, e.a.width);
    const int lacks = lacking(e.a, e.a.table, e.from, pages_wanted(e.length, e.a.page_shift, e.a.width), 0, first);
    const int held = resize_columns<true>(e.a, 0, e.from, e.a.width, 0, e.free, e.a.list, e.length, 0, first);
    if (lane_id() == 0) e.said[0] = lacks, e.said[1] = held;
}

}  // namespace
}  // namespace w4g64

// `table` and `new_table`: the columns from `from` on of a row of `width`.
extern "C" void ends_resize(const int32_t* table, int32_t* new_table, int32_t* new_users, int32_t* list, int32_t* said,
                            int64_t width, int64_t from, int pages, int free, int length, int page_shift) {
    using namespace w4g64;
    EndsArgs e{};
    e.a.table = table - from, e.a.new_table = new_table - from, e.a.new_users = new_users, e.a.list = list;
    e.a.batch = 1, e.a.width = (int)width, e.a.pages = pages, e.a.page_shift = page_shift;
    e.from = (uint32_t)from, e.free = free, e.length = length, e.said = said;
    hipLaunchKernelGGL(ends_kernel, dim3(1), dim3(64), 0, nullptr, e);
}
