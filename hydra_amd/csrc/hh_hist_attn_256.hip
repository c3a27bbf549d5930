// hh_hist_attn_256.hip — the kernels of hh_hist_attn.hpp for heads of 256.
#include "hh_hist_attn.hpp"

namespace hh {
template hipError_t launch_history_attention_d<256>(HistAttnArgs, int, hipStream_t, int *);
}
