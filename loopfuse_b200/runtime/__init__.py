from .kv_pool import KVPool, KVState
from .kv_pool_q4 import QuantKVPool
from .executor import AgentExecutor, ExecutionResult, StepTrace
