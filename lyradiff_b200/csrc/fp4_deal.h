// How the few-row FP4 kernel deals the K blocks of a CTA to the four warps that quantize X.  Plain C++, so that the order can be checked without a GPU.
//
// A quarter of a warp has a row's 256 values of a K block.  Up to four rows, a warp has quarters for 4 / rows K blocks at a time (rows in powers of
// two); more rows take two or four warps for one K block.  K block i of a CTA uses stage i % stages of the ring, for the (i / stages)-th time.  The wait
// for a stage is by the parity of its barrier's phase and tells a phase from the one before it, no more: a warp that skipped one would pass too
// early.  So the warps that share a K block take every kDealWarps / warps_per_kb-th one, also within what they hold at a time: a stage of theirs is theirs every time.
#pragma once

#ifdef __CUDACC__
#define LYRAQ_DEAL_FN __host__ __device__ inline
#else
#define LYRAQ_DEAL_FN inline
#endif

namespace lyraq {
namespace fp4 {

constexpr int kDealWarps  = 4;
constexpr int kDealStages = 4;
static_assert(kDealStages % kDealWarps == 0, "the warps of a stage are the same every time");

struct FewRowsDeal {
    int rows_log2;       // rows, up to the next power of two
    int per_visit;       // K blocks that a warp holds at a time
    int warps_per_kb;
    int step;            // from one of its K blocks to the next: kDealWarps / warps_per_kb
};

LYRAQ_DEAL_FN FewRowsDeal few_rows_deal(int rows)
{
    FewRowsDeal d{0, 1, 1, 0};
    while (1 << d.rows_log2 < rows) {
        ++d.rows_log2;
    }
    if (d.rows_log2 <= 2) {
        d.per_visit = 4 >> d.rows_log2;
    } else {
        d.warps_per_kb = 1 << (d.rows_log2 - 2);
    }
    d.step = kDealWarps / d.warps_per_kb;
    return d;
}

// K block of a CTA that a warp has in the piece-th place of a visit
LYRAQ_DEAL_FN int few_rows_block(const FewRowsDeal& d, int warp, int visit, int piece)
{
    return warp / d.warps_per_kb + d.step * (visit * d.per_visit + piece);
}

}  // namespace fp4
}  // namespace lyraq
