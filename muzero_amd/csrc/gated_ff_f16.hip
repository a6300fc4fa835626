// The gated feed-forward operator's kernels for IEEE half operands (gated_ff.h).
#define MZ_GFF_KERNELS
#include "gated_ff.h"

namespace mz_gff {
int launch_f16(const Args& a, int mode, int tile, hipStream_t s) { return launch_any<_Float16>(a, mode, tile, s); }
int launch_both_f16(const Args& x, const Args& w, int tile, hipStream_t s) { return launch_both<_Float16>(x, w, tile, s); }
int launch_few_f16(const Args& a, hipStream_t s) { return launch_few<_Float16>(a, s); }
}  // namespace mz_gff
