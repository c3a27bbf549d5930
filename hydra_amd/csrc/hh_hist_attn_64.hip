// hh_hist_attn_64.hip — the kernels of hh_hist_attn.hpp for heads of 64.
#include "hh_hist_attn.hpp"

namespace hh {
template hipError_t launch_history_attention_d<64>(HistAttnArgs, int, hipStream_t, int *);
}
