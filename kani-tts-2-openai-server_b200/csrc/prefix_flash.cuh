// The tensor-core attention over a shared prefix (and, in the prompt pass, each
// stream's own rows) that both entry points launch; kernels in prefix_prefill.cu.
#pragma once

#include "prefix_attn.cuh"

namespace kani {
namespace prefix {

// Splits of `rows` K / V rows over CTAs, for batch x tokens x hq query rows.
int flash_splits(int64_t batch, int64_t tokens, int hq, int hk, int64_t rows);

// One launch.  own_rows: with the streams' own rows (the prompt pass), else the prefix
// alone, of all of batch x tokens queries.  ml / acc: partials [splits][rows][2] and
// [splits][rows][D] (fp32; maximum in powers of 2, sum, unnormalised output; a sum of
// 0 = no row seen); NULL (one split only): the result goes to p.out.
int launch_flash(const Params& p, int32_t dtype, int d, int batch, int tokens, bool own_rows, int splits, float* ml,
                 float* acc, bool dependent, cudaStream_t s);

}  // namespace prefix
}  // namespace kani
