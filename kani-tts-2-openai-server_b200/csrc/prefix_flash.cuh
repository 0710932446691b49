// The tensor-core attention over a shared prefix (and, in the prompt pass, each
// stream's own rows) that both entry points launch; kernels in prefix_prefill.cu.
#pragma once

#include "prefix_attn.cuh"

namespace kani {
namespace prefix {

// How the K / V rows of each 128 queries of a KV head are split over CTAs: `parts`
// clusters of `cluster` CTAs, whose results the cluster joins.
struct FlashSplit {
  int cluster, parts;
};
FlashSplit flash_split(int64_t batch, int64_t tokens, int hq, int hk, int64_t rows, int most_parts);

// One launch.  own_rows: with the streams' own rows (the prompt pass), else the prefix
// alone, of all of batch x tokens queries.  ml / acc: partials [parts][rows][2] and
// [parts][rows][D] (fp32; maximum in powers of 2, sum, unnormalised output; a sum of
// 0 = no row seen, with an output of zeros); NULL (one part only): the result goes to
// p.out.  dependent: as a programmatic dependent of the launch before it.
int launch_flash(const Params& p, int32_t dtype, int d, int batch, int tokens, bool own_rows, FlashSplit split,
                 float* ml, float* acc, bool dependent, cudaStream_t s);

}  // namespace prefix
}  // namespace kani
