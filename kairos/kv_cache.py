from kairos_amd.kv_cache import *  # noqa: F401,F403
from kairos_amd import kv_cache as _impl

globals().update({k: v for k, v in vars(_impl).items() if not k.startswith("__")})
