// esda_internal.h -- library-internal hooks shared by the HIP sources and the ES* C++
// layer (not part of the public ABI).
#pragma once
#include <string>

struct ihipStream_t;
struct esda_prefix_desc;
struct esda_prefix_args;

namespace esda_detail {
// Sets the calling thread's esda_last_error() message.
void set_error(const std::string &msg);
// ESDA_OK when the current device is a gfx950; otherwise sets the message and returns
// ESDA_ERR_DEVICE or ESDA_ERR_HIP.
int check_device();
// The prefix part of esda_prefix_decode (esda_prefix_tiles.hip): the key splits of its plan, or
// what is wrong with the description; and its launch, which returns a hipError_t.
const char *prefix_tiles_plan(const esda_prefix_desc *d, int *splits);
int prefix_tiles(const esda_prefix_desc *d, const esda_prefix_args *a, float *part_acc, float *part_ml, ihipStream_t *st);
}  // namespace esda_detail
