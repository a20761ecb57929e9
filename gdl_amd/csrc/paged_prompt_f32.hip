// paged_prompt_f32.hip — float32 queries over paged caches.
#include "paged_prompt.hpp"

namespace geo {
namespace paged {
template int prompt_of<float>(int, const Prompt&, const PromptPlan&, void*, float*, hipStream_t);
}  // namespace paged
}  // namespace geo
