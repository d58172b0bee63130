// tensors.cpp — the host side of calls that take whole lists of tensors (liftreg_amd/optim.py): checks and addresses of every
// tensor of several parallel lists in one call.  In Python the same checks cost about 0.3 us a tensor, which for the 18 tensors of
// the network is three times what the kernel takes.  Loaded with ctypes.PyDLL (the interpreter's lock is held); host code only.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

namespace {

bool is_kind(char kind, at::ScalarType t, at::ScalarType first) {
  switch (kind) {
    case 'p': return t == first;                    // the first list's type: float32 or bfloat16
    case 'f': return t == at::kFloat;
    case 'm': return t == at::kFloat8_e4m3fn;
    case 'v': return t == at::kFloat8_e5m2;
    case 's': return t == at::kFloat8_e8m0fnu;      // one for each 32 elements of the first list's tensor
    default: return false;
  }
}

}  // namespace

// lists: a tuple of lists of n tensors each, kinds: a character for each list (above).  Writes the addresses, list after list, then
// the n sizes of the first list's tensors to out (room for `room` numbers) and info = {device index, 1 if bfloat16}.  Returns n, or
// -1 if anything is not as it must be: a list's length, a type, a device, a size, a tensor that is not contiguous, an address that
// occurs twice in the lists that are written (all but kind 'p' of index `read_only`).  The caller then finds out what it is.
extern "C" int64_t lr_gather_tensors(PyObject* lists, const char* kinds, int read_only, uint64_t* out, int64_t room, int32_t* info) {
  try {
    if (!PyTuple_CheckExact(lists)) return -1;
    const int64_t k = PyTuple_GET_SIZE(lists);
    int64_t n = -1;
    at::ScalarType first = at::kFloat;
    at::DeviceIndex device = -1;
    std::vector<uint64_t> written;
    for (int64_t j = 0; j < k; ++j) {
      PyObject* list = PyTuple_GET_ITEM(lists, j);
      if (!kinds[j] || !PyList_CheckExact(list)) return -1;
      if (j == 0) {
        n = PyList_GET_SIZE(list);
        if (n < 1 || (k + 1) * n > room) return -1;
        written.reserve(static_cast<size_t>(k * n));
      }
      if (PyList_GET_SIZE(list) != n) return -1;
      for (int64_t i = 0; i < n; ++i) {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) return -1;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || !t.device().is_cuda() || t.layout() != at::kStrided) return -1;
        if (j == 0 && i == 0) {
          first = t.scalar_type();
          device = t.device().index();
          if (first != at::kFloat && first != at::kBFloat16) return -1;
        }
        const int64_t size = j == 0 ? t.numel() : static_cast<int64_t>(out[k * n + i]);
        if (t.device().index() != device || !is_kind(kinds[j], t.scalar_type(), first) || !t.is_contiguous() ||
            t.numel() != (kinds[j] == 's' ? (size + 31) / 32 : size))
          return -1;
        const uint64_t at = reinterpret_cast<uint64_t>(t.data_ptr());
        out[j * n + i] = at;
        if (j == 0) out[k * n + i] = static_cast<uint64_t>(size);
        if (j != read_only && size) written.push_back(at);
      }
    }
    std::sort(written.begin(), written.end());
    if (std::adjacent_find(written.begin(), written.end()) != written.end()) return -1;
    info[0] = device;
    info[1] = first == at::kBFloat16;
    return n;
  } catch (...) {
    return -1;
  }
}
