// The places of the packed attention's workgroups alone: which tile of which sequence
// each one takes.
#include "qwen2_packed_attention.hip"

namespace w4g64 {
namespace {

struct FindsArgs {
    PackedArgs a;
    int longest;
    int32_t* said;  // of each workgroup: found, begin, count, tile, head
};

template <int kRows>
void finds_kernel(FindsArgs f) {
    Piece s{-1, -1, -1, -1};
    const int item = (int)blockIdx.x, lane = (int)threadIdx.x;
    const bool found = f.longest == 2   ? find_longest<kRows, true>(f.a, item, lane, s)
                       : f.longest == 1 ? find_longest<kRows, false>(f.a, item, lane, s)
                                        : find_in_turn<kRows>(f.a, item, lane, s);
    const int said[5] = {found, s.begin, s.count, s.tile, s.kvh};
    if (lane < 5) f.said[5 * item + lane] = said[lane];
}

}  // namespace
}  // namespace w4g64

extern "C" void finds(const int32_t* cu_rows, int32_t* said, int batch, int rows, int group, int kv_heads, int tile_rows,
                      int longest, int workgroups) {
    using namespace w4g64;
    FindsArgs f{};
    f.a.cu_rows = cu_rows, f.a.batch = batch, f.a.rows = rows, f.a.group = group, f.a.kv_heads = kv_heads;
    f.a.heads = group * kv_heads, f.a.by_group = divisor(group), f.a.by_kv_heads = divisor(kv_heads);
    f.longest = longest, f.said = said;
    const dim3 grid((unsigned)workgroups);
    if (tile_rows == 32) hipLaunchKernelGGL(finds_kernel<32>, grid, dim3(64), 0, nullptr, f);
    else if (tile_rows == 64) hipLaunchKernelGGL(finds_kernel<64>, grid, dim3(64), 0, nullptr, f);
    else hipLaunchKernelGGL(finds_kernel<128>, grid, dim3(64), 0, nullptr, f);
}
