"""B200-native Mamba-2 SSD operator behind the trading_bot_0 operator surface."""
from . import _lib
from .ssd import (alloc_workspace, backward, forward, make_dims, ssd_scan, state_update, workspace_bytes)
from .stream import StreamState, init_stream_state_batched
from . import sp
from .linear import linear_backward, linear_forward
from .selective import selective_scan, selective_scan_backward, selective_scan_forward, selective_step
from .mixer import mamba2_mixer, mamba2_mixer_step, selective_mixer, selective_mixer_step
from . import linear  # noqa: F401  (the module; its differentiable call is linear.linear)

__all__ = ["forward", "backward", "state_update", "ssd_scan", "make_dims", "workspace_bytes",
           "alloc_workspace", "StreamState", "init_stream_state_batched", "_lib",
           "selective_scan", "selective_scan_forward", "selective_scan_backward", "selective_step", "linear_forward",
           "linear_backward", "mamba2_mixer", "mamba2_mixer_step", "selective_mixer", "selective_mixer_step"]
