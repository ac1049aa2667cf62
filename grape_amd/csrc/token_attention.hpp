// The single tokens' attention, as the attention of several tokens calls it.
#pragma once
#include "common.hpp"

namespace grape {

int attend_single(const grape_wit_window_attention_args& args, const grape_wit_cache& cache, grape_stream_t stream);

}  // namespace grape
