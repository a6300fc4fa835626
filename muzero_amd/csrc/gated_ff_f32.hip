// The gated feed-forward operator's kernels for float32 operands (gated_ff.h).
#define MZ_GFF_KERNELS
#include "gated_ff.h"

namespace mz_gff {
int launch_f32(const Args& a, int mode, int tile, hipStream_t s) { return launch_any<float>(a, mode, tile, s); }
int launch_both_f32(const Args& x, const Args& w, int tile, hipStream_t s) { return launch_both<float>(x, w, tile, s); }
int launch_few_f32(const Args& a, hipStream_t s) { return launch_few<float>(a, s); }
}  // namespace mz_gff
