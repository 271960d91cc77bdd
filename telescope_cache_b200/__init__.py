"""B200-native (sm_100a) telescoping multiresolution attention.

``telescope_cache_b200.reference`` mirrors the reference's ``reference.py``
API; ``telescope_cache_b200.range_spec`` its integer schedule; and
``telescope_cache_b200.telescoping_attn.*`` its split modules.  Next to them
are the operators of the layers that a hybrid stack keeps at full attention:
rotary positions, packed causal attention and the 8-bit key / value cache.  All compute
runs in ``_lib/libtelescope_b200.so`` (CUDA, sm_100a) through a C ABI
(``include/telescope_cache.h``).
"""

from . import range_spec  # noqa: F401
from .reference import *  # noqa: F401,F403
from .reference import __all__  # noqa: F401
from .telescoping_attn.causal import Segments, causal_attention, causal_attention_backward, segment_bounds  # noqa: F401
from .telescoping_attn.kv_cache import (KVCache, cached_attention, cached_attention_step, init_kv_cache,  # noqa: F401
                                        read_kv_cache, write_kv_cache)
from .telescoping_attn.rotary import rotary, rotary_tables  # noqa: F401
