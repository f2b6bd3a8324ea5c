"""The native binding of the cached-decoding operators (``_decode.so``).

Its functions check their arguments, allocate the outputs and launch on the
current stream of the tensors' device, all natively: a decoding step's calls
take a few microseconds on the device, so a wrapper's own time is the call's.
"""

import torch  # noqa: F401  (its libraries are the binding's)

from voyager_b200 import _lib

_lib.load()
try:
    from voyager_b200 import _decode as native
except ImportError as e:
    raise ImportError("voyager_b200/_decode.so is missing or does not fit this torch: build it with "
                      "`python -c 'import __graft_entry__ as g; g.build()'`") from e

native.bind(_lib.check)
