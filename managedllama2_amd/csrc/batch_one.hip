// Products of a step of one token: the int4 mat-vec kernel of a decode step (int4_kernels.hpp), with the token's position, its adapter's part
// and a residual in its epilogue.  What the adapter's ranks received comes from the launch in front, as for few tokens (batch_product.hip).
//
// HBM and latency bound them.  Against the tiles of batch_product.hip, of whose 16 rows one token uses one: 4096 columns of 4096 inputs 5.7 -> 3.6 us,
// with an adapter of 16 ranks 9.0 -> 6.9; three of them 10.7 -> 7.3, with 64 ranks 15.5 -> 10.9; gated 2 * 11008 14.7 -> 9.9, with 16 ranks 18.9 -> 13.2;
// 5120 columns of 13824 inputs 13.8 -> 11.0; 32000 columns the same.  Tensors of different widths stay with the tiles, which take them in one
// launch (4096 + 1024 + 1024 columns 7.0 us).  Three tensors of 8193 .. 10240 inputs are short of 4 registers (20 bytes of scratch per lane).
//
// The kernel sums up x w and z x apart for every 32 inputs, in fp32: exact integers of up to 15 where the tiles have differences, so that
// its error grows with |x| (w + z) s.
#include "batch_product.hpp"
#include "int4_kernels.hpp"

namespace l2 {

template <int MODE>
static bool launch_one(const OneTokenArgs& a)
{
    switch (chunk_columns(a.ws)) {
    case 1: return launch_span<1, MODE, STAGE_X>(a);
    case 2: return launch_span<2, MODE, STAGE_X>(a);
    case 3: return launch_span<3, MODE, STAGE_X>(a);
    case 4: return launch_span<4, MODE, STAGE_X>(a);
    case 5: return launch_span<5, MODE, STAGE_X>(a);
    case 6: return launch_span<6, MODE, STAGE_X>(a);
    case 7: return launch_span<7, MODE, STAGE_X>(a);
    default: return false; // beyond 14336 inputs the registers of two or three tensors do not suffice
    }
}

bool launch_one_token(const ProductArgs& call, int n_matrices, bool gated)
{
    if (n_matrices != 1 && n_matrices != (gated ? 2 : 3))
        return false;
    OneTokenArgs a{};
    for (int i = 0; i < n_matrices; ++i) {
        const ProductTensor& t = call.t[i];
        if (t.cols != call.t[0].cols)
            return false;
        a.m[i] = QW{t.w, t.z, t.s};
        a.out[i] = t.out;
        a.residual[i] = t.residual;
        a.part[i] = {t.up, static_cast<const float*>(t.low), t.info ? &t.info->rank : nullptr, t.up_stride, t.n_adapters, t.max_rank};
    }
    a.x = call.x;
    a.K = call.K, a.N = call.t[0].cols, a.ws = weight_words(call.K), a.ss = weight_groups(call.K), a.zs = zero_words(call.K);
    a.n_tensors = gated ? 1 : n_matrices;
    a.positions = call.positions, a.token_adapters = call.token_adapters, a.most_adapters = call.most_adapters;
    return gated ? launch_one<ONE_GATED>(a) : launch_one<ONE_ROWS>(a);
}

} // namespace l2
