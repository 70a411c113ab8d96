from .attn_shared import attn_shared, attn_shared_check
from .lib import BODY, EtxbError, StepParams, build, check, device_info, load
from .pages import PagePool, copy_pages
from .sampling import Sampled, Sampling, sample
from .session import ExchangeRegion, Session, attn_fused_static, op_launch

__all__ = ["BODY", "EtxbError", "StepParams", "build", "check", "device_info", "load", "ExchangeRegion", "Session", "attn_fused_static", "op_launch",
           "attn_shared", "attn_shared_check", "PagePool", "copy_pages", "Sampled", "Sampling", "sample"]
