// The gated feed-forward operator's kernels for bf16 operands (gated_ff.h).
#define MZ_GFF_KERNELS
#include "gated_ff.h"

namespace mz_gff {
int launch_bf16(const Args& a, int mode, int tile, hipStream_t s) { return launch_any<__bf16>(a, mode, tile, s); }
int launch_both_bf16(const Args& x, const Args& w, int tile, hipStream_t s) { return launch_both<__bf16>(x, w, tile, s); }
int launch_few_bf16(const Args& a, hipStream_t s) { return launch_few<__bf16>(a, s); }
}  // namespace mz_gff
