// forms.cpp — the form of a call's tensors for a Python binding (tsn_form_take): what a call's checks went by, compared
// in one call from Python. Seven tensors take 1.1 us, through their attributes 3.3 us: a norm of two rows, bound by its
// call, went from 7.5 to 4.7 us.
#include "../../include/tsn.h"

#include <cstring>

namespace {

// DLPack's view of a tensor (a published C interface; its structure of ABI version 1)
struct View {
    void * data;
    int32_t device_type, device;
    int32_t ndim;
    uint32_t dtype;   // code and bits in 8 bits each, lanes in 16
    int64_t * shape, * strides;
    uint64_t byte_offset;
};
static_assert(sizeof(View) == 48, "the view's layout");

struct Head {   // of a Python object
    intptr_t count;
    void * type;
};

} // namespace

extern "C" int tsn_form_take(tsn_form * f, int record, void * tuple) {
    if (!f || f->n > TSN_FORM_TENSORS) return 0;
    const bool known = f->valid && !record;
    f->valid = 0;   // until every tensor has been found in its form
    if (!known && !record) return 0;
    for (uint32_t i = 0; i < f->n; ++i) {
        tsn_form_tensor & t = f->t[i];
        void * const object = f->item(tuple, i);
        if (!object) return 0;
        const int there = object != f->none;
        if (known && there != t.there) return 0;
        t.there = there;
        if (!there) {
            *f->to[i] = nullptr;
            continue;
        }
        View v;
        memset(&v, 0, sizeof v);
        if (((const Head *) object)->type != f->type || f->view(object, &v) != 0 || v.ndim < 0 || v.ndim > 4 || !v.strides) return 0;
        const size_t bytes = (size_t) v.ndim * 8;
        if (record) {
            t.device_type = v.device_type; t.device = v.device; t.ndim = v.ndim; t.dtype = v.dtype;
            memcpy(t.shape, v.shape, bytes);
            memcpy(t.strides, v.strides, bytes);
        } else if (t.device_type != v.device_type || t.device != v.device || t.ndim != v.ndim || t.dtype != v.dtype ||
                   memcmp(t.shape, v.shape, bytes) != 0 || memcmp(t.strides, v.strides, bytes) != 0) {
            return 0;
        }
        *f->to[i] = (char *) v.data + v.byte_offset;
    }
    f->valid = 1;
    return 1;
}
