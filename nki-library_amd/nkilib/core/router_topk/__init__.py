from .router_topk import route_for_moe, router_topk
from .router_topk_bwd import router_topk_bwd

__all__ = ["router_topk", "route_for_moe", "router_topk_bwd"]
