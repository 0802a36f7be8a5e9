from .compressed_linear import *  # noqa: F401,F403
from .packed import packed_linear  # noqa: F401
