"""Hand-written sm_100a kernels and their Python entry points."""

from .functions import *  # noqa: F401,F403
from .functions import __all__ as _functions
from .fp8 import *  # noqa: F401,F403
from .fp8 import __all__ as _fp8
from .int8 import *  # noqa: F401,F403
from .int8 import __all__ as _int8
from .logprobs import *  # noqa: F401,F403
from .logprobs import __all__ as _logprobs

__all__ = [*_functions, *_fp8, *_int8, *_logprobs]
