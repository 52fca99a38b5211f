// The kernels of miq_paged_attention (attention_paged.h) of fp32 caches.
#include "attention_paged.h"

namespace miq {

int paged_attention_f32(const PagedCall& a) { return paged_attention_cache<float>(a); }

}  // namespace miq
