// GENERATED by dart/lib/cuda/gen_fml_bindings.py from include/fml.h -- do not edit by hand.
// dart:ffi binding of libflutter_ml_b200.so: every struct, constant and entry point of the C ABI.
// Replaces the two typedefs and the single lookup of the original lib/cuda/cudacaller.dart.
// ignore_for_file: non_constant_identifier_names, constant_identifier_names
import 'dart:ffi';

import 'package:ffi/ffi.dart';

/// Opaque `fml_ctx` handle.
final class FmlCtx extends Opaque {}

/// `fml_status`.
abstract final class FmlStatus {
  static const int FML_OK = 0;
  static const int FML_ERR_INVALID = -1;
  static const int FML_ERR_CUDA = -2;
  static const int FML_ERR_NO_DEVICE = -3;
  static const int FML_ERR_TIMEOUT = -4;
  static const int FML_ERR_NCCL = -5;
  static const int FML_ERR_OOM = -6;
}

/// `fml_precision`.
abstract final class FmlPrecision {
  static const int FML_PREC_TF32 = 0;
  static const int FML_PREC_3XTF32 = 1;
  static const int FML_PREC_FP32 = 2;
}

/// `fml_act`.
abstract final class FmlAct {
  static const int FML_ACT_NONE = 0;
  static const int FML_ACT_RELU = 1;
  static const int FML_ACT_SIGMOID = 2;
  static const int FML_ACT_TANH = 3;
  static const int FML_ACT_GELU = 4;
}

/// `fml_optimizer`.
abstract final class FmlOptimizer {
  static const int FML_OPT_MOMENTUM = 1;
  static const int FML_OPT_NAG = 2;
  static const int FML_OPT_RMSPROP = 3;
  static const int FML_OPT_ADAGRAD = 4;
  static const int FML_OPT_ADAMW = 6;
  static const int FML_OPT_AMSGRAD = 7;
}

/// `fml_act2`.
abstract final class FmlAct2 {
  static const int FML_ACT2_LEAKY_RELU = 5;
  static const int FML_ACT2_ELU = 6;
  static const int FML_ACT2_SWISH = 7;
  static const int FML_ACT2_MISH = 8;
}

/// `fml_op_kind`.
abstract final class FmlOpKind {
  static const int FML_OP_MATMUL = 1;
  static const int FML_OP_MATVECMUL = 2;
  static const int FML_OP_ADD_MATRIX_AND_VECTOR = 3;
  static const int FML_OP_ADD = 4;
  static const int FML_OP_MULTIPLY = 5;
  static const int FML_OP_RELU = 6;
  static const int FML_OP_SIGMOID = 7;
  static const int FML_OP_TANH = 8;
  static const int FML_OP_GELU = 9;
  static const int FML_OP_LEAKY_RELU = 10;
  static const int FML_OP_ELU = 11;
  static const int FML_OP_SWISH = 12;
  static const int FML_OP_MISH = 13;
  static const int FML_OP_SCALE_MATRIX = 14;
  static const int FML_OP_TRANSPOSE = 15;
  static const int FML_OP_CONCAT = 16;
  static const int FML_OP_SOFTMAX_MATRIX = 17;
  static const int FML_OP_LAYER_NORM = 18;
  static const int FML_OP_EMBEDDING_LOOKUP = 19;
  static const int FML_OP_MSE = 20;
  static const int FML_OP_SUM = 21;
  static const int FML_OP_SOFTMAX_XENT = 22;
  static const int FML_OP_DENSE = 23;
  static const int FML_OP_CONV2D = 24;
  static const int FML_OP_ADD_SCALAR_TO_MATRIX = 25;
  static const int FML_OP_ATTENTION = 26;
}

/// `fml_tape_direction`.
abstract final class FmlTapeDirection {
  static const int FML_TAPE_FORWARD = 0;
  static const int FML_TAPE_BACKWARD = 1;
  static const int FML_TAPE_BACKWARD_NOSEED = 2;
}

/// `fml_recurrence_form`.
abstract final class FmlRecurrenceForm {
  static const int FML_RECURRENCE_GATED = 0;
  static const int FML_RECURRENCE_LINEAR = 1;
}

abstract final class FmlLimits {
  static const int FML_XENT_STATIC_MAX_ROWS = 65536;
  static const int FML_QK_NORM_ROPE_PARTS = 592;
}

/// `fml_config` of include/fml.h (16 bytes).
final class FmlConfig extends Struct {
  @Int32() external int device;
  @Int32() external int precision;
  @Int64() external int workspaceBytes;
}

/// `fml_gemm_desc` of include/fml.h (200 bytes).
final class FmlGemmDesc extends Struct {
  @Int32() external int M;
  @Int32() external int N;
  @Int32() external int K;
  @Int32() external int transA;
  @Int32() external int transB;
  @Int64() external int lda;
  @Int64() external int ldb;
  @Int64() external int ldc;
  external Pointer<Float> A;
  external Pointer<Float> B;
  external Pointer<Float> C;
  external Pointer<Float> bias;
  external Pointer<Float> preact;
  @Int32() external int act;
  @Float() external double alpha;
  @Float() external double beta;
  @Int32() external int batch1;
  @Int32() external int batch2;
  @Int64() external int sA1;
  @Int64() external int sA2;
  @Int64() external int sB1;
  @Int64() external int sB2;
  @Int64() external int sC1;
  @Int64() external int sC2;
  @Int32() external int precision;
  external Pointer<Float> dactSaved;
  @Int32() external int dact;
  @Int32() external int rowop;
  @Int32() external int rowopCausal;
  external Pointer<Float> rowopAux;
}

/// `fml_op` of include/fml.h (144 bytes).
final class FmlOp extends Struct {
  @Int32() external int kind;
  @Int32() external int rows;
  @Int32() external int cols;
  @Int32() external int inner;
  @Array(3) external Array<Pointer<Float>> inp;
  @Array(3) external Array<Pointer<Float>> gin;
  external Pointer<Float> out;
  external Pointer<Float> gout;
  @Array(2) external Array<Pointer<Float>> aux;
  external Pointer<Int32> ids;
  external Pointer<Pointer<Float>> parts;
  external Pointer<Pointer<Float>> gparts;
  external Pointer<Int32> partCols;
  @Int32() external int nParts;
  @Float() external double s;
  @Int32() external int iparam;
  @Int32() external int precision;
}

/// `fml_attention_desc` of include/fml.h (80 bytes).
final class FmlAttentionDesc extends Struct {
  @Int32() external int nSeq;
  @Int32() external int seqLen;
  @Int32() external int heads;
  @Int32() external int dHead;
  external Pointer<Float> q;
  external Pointer<Float> k;
  external Pointer<Float> v;
  @Int64() external int ldQkv;
  external Pointer<Float> out;
  @Int64() external int ldOut;
  external Pointer<Float> lse;
  @Float() external double scale;
  @Int32() external int causal;
}

/// `fml_lstm_desc` of include/fml.h (72 bytes).
final class FmlLstmDesc extends Struct {
  @Int32() external int T;
  @Int32() external int B;
  @Int32() external int I;
  @Int32() external int H;
  external Pointer<Float> W;
  external Pointer<Float> b;
  external Pointer<Float> x;
  external Pointer<Float> gates;
  external Pointer<Float> cells;
  external Pointer<Float> hs;
  external Pointer<Float> xproj;
}

/// One field per entry point; `FmlBindings(DynamicLibrary.open('cuda_lib/libflutter_ml_b200.so'))`.
class FmlBindings {
  final DynamicLibrary lib;
  FmlBindings(this.lib);

  late final fmlInit = lib.lookupFunction<
      Int32 Function(Pointer<FmlConfig>, Pointer<Pointer<FmlCtx>>),
      int Function(Pointer<FmlConfig>, Pointer<Pointer<FmlCtx>>)>('fml_init');
  late final fmlShutdown = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_shutdown');
  late final fmlLastError = lib.lookupFunction<
      Pointer<Utf8> Function(Pointer<FmlCtx>),
      Pointer<Utf8> Function(Pointer<FmlCtx>)>('fml_last_error');
  late final fmlDeviceCount = lib.lookupFunction<
      Int32 Function(Pointer<Int32>),
      int Function(Pointer<Int32>)>('fml_device_count');
  late final fmlDeviceName = lib.lookupFunction<
      Int32 Function(Int32, Pointer<Utf8>, Int32),
      int Function(int, Pointer<Utf8>, int)>('fml_device_name');
  late final fmlSmCount = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, Pointer<Int32>)>('fml_sm_count');
  late final fmlSetSmReserve = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_set_sm_reserve');
  late final fmlSetStream = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Void>),
      int Function(Pointer<FmlCtx>, Pointer<Void>)>('fml_set_stream');
  late final fmlSync = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_sync');
  late final fmlDeviceStatus = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, Pointer<Int32>)>('fml_device_status');
  late final fmlSelftestWaitTimeout = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_selftest_wait_timeout');
  late final fmlSelftestClusterWait = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32),
      int Function(Pointer<FmlCtx>, int, int)>('fml_selftest_cluster_wait');
  late final fmlSelftestPerDeviceOnce = lib.lookupFunction<
      Int32 Function(Int32, Pointer<Int32>),
      int Function(int, Pointer<Int32>)>('fml_selftest_per_device_once');
  late final fmlAlloc = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int64, Pointer<Pointer<Float>>),
      int Function(Pointer<FmlCtx>, int, Pointer<Pointer<Float>>)>('fml_alloc');
  late final fmlMemInfo = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int64>, Pointer<Int64>, Pointer<Int64>),
      int Function(Pointer<FmlCtx>, Pointer<Int64>, Pointer<Int64>, Pointer<Int64>)>('fml_mem_info');
  late final fmlFree = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<Float>)>('fml_free');
  late final fmlZero = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int)>('fml_zero');
  late final fmlFill = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int64, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int, double)>('fml_fill');
  late final fmlUploadF32 = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int)>('fml_upload_f32');
  late final fmlUploadF64 = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Double>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Double>, int)>('fml_upload_f64');
  late final fmlUploadI32 = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>, Pointer<Int32>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Int32>, Pointer<Int32>, int)>('fml_upload_i32');
  late final fmlDownloadF32 = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int)>('fml_download_f32');
  late final fmlDownloadF64 = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Double>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Double>, Pointer<Float>, int)>('fml_download_f64');
  late final fmlCopy = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int)>('fml_copy');
  late final fmlHostAlloc = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int64, Pointer<Pointer<Void>>),
      int Function(Pointer<FmlCtx>, int, Pointer<Pointer<Void>>)>('fml_host_alloc');
  late final fmlHostFree = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Void>),
      int Function(Pointer<FmlCtx>, Pointer<Void>)>('fml_host_free');
  late final fmlStageRows = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Void>, Pointer<Void>, Int32, Int64, Pointer<Int64>, Int64, Int64, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Void>, Pointer<Void>, int, int, Pointer<Int64>, int, int, int)>('fml_stage_rows');
  late final fmlStageRowsAsync = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Void>, Pointer<Void>, Int32, Int64, Pointer<Int64>, Int64, Int64, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Void>, Pointer<Void>, int, int, Pointer<Int64>, int, int, int)>('fml_stage_rows_async');
  late final fmlStageWait = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_stage_wait');
  late final fmlLaneH2d = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, int)>('fml_lane_h2d');
  late final fmlLaneD2h = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, int)>('fml_lane_d2h');
  late final fmlLaneSync = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_lane_sync');
  late final fmlEventRecordOn = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32),
      int Function(Pointer<FmlCtx>, int, int)>('fml_event_record_on');
  late final fmlWaitEvent = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32),
      int Function(Pointer<FmlCtx>, int, int)>('fml_wait_event');
  late final fmlEventSync = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_event_sync');
  late final fmlGraphBegin = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_graph_begin');
  late final fmlGraphEnd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, Pointer<Int32>)>('fml_graph_end');
  late final fmlGraphLaunch = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_graph_launch');
  late final fmlGraphDestroy = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_graph_destroy');
  late final fmlTimerStart = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_timer_start');
  late final fmlTimerStopMs = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<Float>)>('fml_timer_stop_ms');
  late final fmlEventRecord = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_event_record');
  late final fmlEventElapsedMs = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32, Pointer<Float>),
      int Function(Pointer<FmlCtx>, int, int, Pointer<Float>)>('fml_event_elapsed_ms');
  late final fmlGemm = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlGemmDesc>),
      int Function(Pointer<FmlCtx>, Pointer<FmlGemmDesc>)>('fml_gemm');
  late final fmlGemmLastPath = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, Pointer<Int32>)>('fml_gemm_last_path');
  late final fmlGemmLastTile = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Int32>, Pointer<Int32>, Pointer<Int32>, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, Pointer<Int32>, Pointer<Int32>, Pointer<Int32>, Pointer<Int32>)>('fml_gemm_last_tile');
  late final multiplyMatrices = lib.lookupFunction<
      Void Function(Pointer<Float>, Pointer<Float>, Pointer<Float>, Int32, Int32, Int32),
      void Function(Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int)>('multiplyMatrices');
  late final benchtest = lib.lookupFunction<
      Int32 Function(),
      int Function()>('benchtest');
  late final fmlActFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, int)>('fml_act_fwd');
  late final fmlActBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int64, Int32, Pointer<Float>),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int, Pointer<Float>)>('fml_act_bwd');
  late final fmlAdd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int)>('fml_add');
  late final fmlAxpy = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Float, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, double, Pointer<Float>, Pointer<Float>, int)>('fml_axpy');
  late final fmlMul = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int)>('fml_mul');
  late final fmlAddBias = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int)>('fml_add_bias');
  late final fmlColSum = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64, Int64, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int, int, int)>('fml_col_sum');
  late final fmlTranspose = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int, int)>('fml_transpose');
  late final fmlSoftmaxRowsFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int, int, double, int)>('fml_softmax_rows_fwd');
  late final fmlSoftmaxRowsBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, double, int)>('fml_softmax_rows_bwd');
  late final fmlLayernormFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, double)>('fml_layernorm_fwd');
  late final fmlLayernormBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int)>('fml_layernorm_bwd');
  late final fmlSoftmaxXent = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, int, int, double)>('fml_softmax_xent');
  late final fmlSoftmaxXentDbias = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, int, int, double, Pointer<Float>)>('fml_softmax_xent_dbias');
  late final fmlSoftmaxXentStatic = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, Int64, Int32, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, int, int, double)>('fml_softmax_xent_static');
  late final fmlMse = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, double)>('fml_mse');
  late final fmlEmbeddingFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, Int64, Int32, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, int, int, int, int)>('fml_embedding_fwd');
  late final fmlEmbeddingBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Int64, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Int32>, Pointer<Float>, int, int, int)>('fml_embedding_bwd');
  late final fmlPositionalTable = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int, int)>('fml_positional_table');
  late final fmlSgdStep = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Int64, Double, Double),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, int, double, double)>('fml_sgd_step');
  late final fmlAdamStep = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Double, Double, Double, Double, Int32, Double),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, double, double, double, double, int, double)>('fml_adam_step');
  late final fmlAdamStepOn = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Double, Double, Double, Double, Int32, Double, Int32),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, double, double, double, double, int, double, int)>('fml_adam_step_on');
  late final fmlOptimizerStep = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Double, Double, Double, Double, Double, Int32),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, double, double, double, double, double, int)>('fml_optimizer_step');
  late final fmlAdamwStateFloats = lib.lookupFunction<
      Int32 Function(Int32, Pointer<Int64>, Int32, Pointer<Int64>),
      int Function(int, Pointer<Int64>, int, Pointer<Int64>)>('fml_adamw_state_floats');
  late final fmlAdamwPlanCreate = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Pointer<Float>>, Pointer<Pointer<Float>>, Pointer<Int64>, Pointer<Float>, Pointer<Float>, Int32, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, int, Pointer<Pointer<Float>>, Pointer<Pointer<Float>>, Pointer<Int64>, Pointer<Float>, Pointer<Float>, int, Pointer<Int32>)>('fml_adamw_plan_create');
  late final fmlAdamwPlanStep = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32, Double, Double, Double, Double, Double, Int32, Double, Int32, Int64),
      int Function(Pointer<FmlCtx>, int, int, double, double, double, double, double, int, double, int, int)>('fml_adamw_plan_step');
  late final fmlAdamwPlanCount = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Int32>),
      int Function(Pointer<FmlCtx>, int, Pointer<Int32>)>('fml_adamw_plan_count');
  late final fmlAdamwPlanSetCount = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32),
      int Function(Pointer<FmlCtx>, int, int)>('fml_adamw_plan_set_count');
  late final fmlAdamwPlanDestroy = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_adamw_plan_destroy');
  late final fmlAct2Fwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Float, Pointer<Float>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, int, double, Pointer<Float>, Pointer<Float>, int)>('fml_act2_fwd');
  late final fmlAct2Bwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Float, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int32),
      int Function(Pointer<FmlCtx>, int, double, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int)>('fml_act2_bwd');
  late final fmlTapeRun = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlOp>, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<FmlOp>, int, int)>('fml_tape_run');
  late final fmlTapeKind = lib.lookupFunction<
      Int32 Function(Pointer<Utf8>),
      int Function(Pointer<Utf8>)>('fml_tape_kind');
  late final fmlAttentionFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlAttentionDesc>),
      int Function(Pointer<FmlCtx>, Pointer<FmlAttentionDesc>)>('fml_attention_fwd');
  late final fmlAttentionBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlAttentionDesc>, Pointer<Float>, Int64, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int32, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<FmlAttentionDesc>, Pointer<Float>, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, Pointer<Float>)>('fml_attention_bwd');
  late final fmlQkNormRopeFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int64, Pointer<Float>, Int64, Int32, Pointer<Float>, Int64, Pointer<Float>, Int64, Int32, Int64, Int32, Pointer<Float>, Pointer<Float>, Pointer<Int32>, Int32, Int32, Int32, Double, Float),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int, Pointer<Float>, int, int, Pointer<Float>, int, Pointer<Float>, int, int, int, int, Pointer<Float>, Pointer<Float>, Pointer<Int32>, int, int, int, double, double)>('fml_qk_norm_rope_fwd');
  late final fmlQkNormRopeBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int64, Pointer<Float>, Int64, Pointer<Float>, Int64, Int32, Pointer<Float>, Int64, Pointer<Float>, Int64, Pointer<Float>, Int64, Int32, Int64, Int32, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Int32>, Int32, Int32, Int32, Double, Float, Int32, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int, Pointer<Float>, int, Pointer<Float>, int, int, Pointer<Float>, int, Pointer<Float>, int, Pointer<Float>, int, int, int, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Int32>, int, int, int, double, double, int, Pointer<Float>)>('fml_qk_norm_rope_bwd');
  late final fmlConv2dFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int32, Int32, Int32, Int32, Int32, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int, int, int, int, int)>('fml_conv2d_fwd');
  late final fmlConv2dBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int32, Int32, Int32, Int32, Int32, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int, int, int, int, int)>('fml_conv2d_bwd');
  late final fmlCheckpointSave = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Utf8>, Int64, Int32, Pointer<Pointer<Utf8>>, Pointer<Pointer<Float>>, Pointer<Int64>),
      int Function(Pointer<FmlCtx>, Pointer<Utf8>, int, int, Pointer<Pointer<Utf8>>, Pointer<Pointer<Float>>, Pointer<Int64>)>('fml_checkpoint_save');
  late final fmlCheckpointLoad = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Utf8>, Pointer<Int64>, Int32, Pointer<Pointer<Utf8>>, Pointer<Pointer<Float>>, Pointer<Int64>),
      int Function(Pointer<FmlCtx>, Pointer<Utf8>, Pointer<Int64>, int, Pointer<Pointer<Utf8>>, Pointer<Pointer<Float>>, Pointer<Int64>)>('fml_checkpoint_load');
  late final fmlLstmFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlLstmDesc>),
      int Function(Pointer<FmlCtx>, Pointer<FmlLstmDesc>)>('fml_lstm_fwd');
  late final fmlLstmBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<FmlLstmDesc>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>),
      int Function(Pointer<FmlCtx>, Pointer<FmlLstmDesc>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>)>('fml_lstm_bwd');
  late final fmlLstmCellFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int64, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int)>('fml_lstm_cell_fwd');
  late final fmlLstmCellBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int32, Int64, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int, int, int)>('fml_lstm_cell_bwd');
  late final fmlGatedRecurrenceFwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32, Int32, Int32, Pointer<Float>, Pointer<Float>, Int64, Int64, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Int64, Int64, Pointer<Float>),
      int Function(Pointer<FmlCtx>, int, int, int, int, Pointer<Float>, Pointer<Float>, int, int, Pointer<Float>, Pointer<Int32>, Pointer<Float>, int, int, Pointer<Float>)>('fml_gated_recurrence_fwd');
  late final fmlGatedRecurrenceBwd = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Int32, Int32, Int32, Pointer<Float>, Pointer<Float>, Int64, Int64, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, Int64, Int64, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, Int32),
      int Function(Pointer<FmlCtx>, int, int, int, int, Pointer<Float>, Pointer<Float>, int, int, Pointer<Float>, Pointer<Int32>, Pointer<Float>, Pointer<Float>, int, int, Pointer<Float>, Pointer<Float>, Pointer<Float>, Pointer<Float>, int)>('fml_gated_recurrence_bwd');
  late final fmlDpUniqueId = lib.lookupFunction<
      Int32 Function(Pointer<Uint8>),
      int Function(Pointer<Uint8>)>('fml_dp_unique_id');
  late final fmlDpInit = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Uint8>, Int32, Int32),
      int Function(Pointer<FmlCtx>, Pointer<Uint8>, int, int)>('fml_dp_init');
  late final fmlDpSetTimeout = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_dp_set_timeout');
  late final fmlDpSetMaxCtas = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32),
      int Function(Pointer<FmlCtx>, int)>('fml_dp_set_max_ctas');
  late final fmlDpAllreduceSum = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, Pointer<Float>, int)>('fml_dp_allreduce_sum');
  late final fmlDpAllreduceSumOn = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>, Int32, Pointer<Float>, Int64),
      int Function(Pointer<FmlCtx>, int, Pointer<Float>, int)>('fml_dp_allreduce_sum_on');
  late final fmlDpShutdown = lib.lookupFunction<
      Int32 Function(Pointer<FmlCtx>),
      int Function(Pointer<FmlCtx>)>('fml_dp_shutdown');
}
