// paged_prompt_f16.hip — float16 queries over paged caches.
#include "paged_prompt.hpp"

namespace geo {
namespace paged {
template int prompt_of<_Float16>(int, const Prompt&, const PromptPlan&, void*, float*, hipStream_t);
}  // namespace paged
}  // namespace geo
