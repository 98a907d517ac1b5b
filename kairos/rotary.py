from kairos_amd.rotary import *  # noqa: F401,F403
from kairos_amd import rotary as _impl

globals().update({k: v for k, v in vars(_impl).items() if not k.startswith("__")})
