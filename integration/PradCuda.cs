// <auto-generated> by integration/make_bindings.py from include/prad_cuda.h -- do not edit by hand.
// P/Invoke surface of libprad_cuda for ParallelReverseAutoDiff (RMAD double / PRADLite float).
namespace ParallelReverseAutoDiff.RMAD.Cuda
{
    using System;
    using System.Runtime.InteropServices;

    /// <summary>One [DllImport] per function of include/prad_cuda.h.</summary>
    public static class PradCuda
    {
        private const string Lib = "prad_cuda";   // libprad_cuda.so / prad_cuda.dll

        public enum Status
        {
            Ok = 0,
            ErrInvalid = 1,
            ErrShape = 2,
            ErrNotInitialized = 3,
            ErrCuda = 4,
            ErrOom = 5,
            ErrUnsupported = 6,
            ErrComm = 7,
            ErrTimeout = 8,
        }

        public const int PackRows = 1;
        public const int PackCols = 2;

        public enum DType
        {
            F32 = 0,
            F64 = 1,
        }

        public enum Act
        {
            None = 0,
            LeakyRelu = 1,
            Sigmoid = 2,
            Tanh = 3,
            Gelu = 4,
            Relu = 5,
            AmplifiedSigmoid = 6,
        }

        public enum AdamForm
        {
            Rmad = 0,
            Prad = 1,
        }

        public enum Op
        {
            Matmul = 0,
            Add = 1,
            Add3 = 2,
            AddBroadcast = 3,
            Hadamard = 4,
            LeakyRelu = 5,
            Sigmoid = 6,
            Tanh = 7,
            Gelu = 8,
            Softmax = 9,
            Layernorm = 10,
            Scale = 11,
            Transpose = 12,
            Relu = 13,
            AmplifiedSigmoid = 14,
            SineSoftmax = 15,
        }

        public enum TensorOp
        {
            Exp = 0,
            Ln = 1,
            Log10 = 2,
            Abs = 3,
            Square = 4,
            Sqrt = 5,
            Sin = 6,
            Cos = 7,
            Reciprocal = 8,
            Negate = 9,
            Add = 16,
            Sub = 17,
            Mul = 18,
            Div = 19,
        }

        public const int StaticColsumMaxCols = 32768;
        public const int ConvMaxWidth = 8;
        public const int DpMarks = 256;

        [StructLayout(LayoutKind.Sequential, CharSet = CharSet.Ansi)]
        public struct DeviceInfo
        {
            public int Device, SmCount, CcMajor, CcMinor, L2Bytes, SmemPerBlockOptin, SmClockKhz, MemClockKhz;
            public ulong TotalBytes, FreeBytes, ScratchBytes;
            [MarshalAs(UnmanagedType.ByValTStr, SizeConst = 64)] public string Name;
        }

        [StructLayout(LayoutKind.Sequential, CharSet = CharSet.Ansi)]
        public struct Timing
        {
            [MarshalAs(UnmanagedType.ByValTStr, SizeConst = 48)] public string Label;
            public double Milliseconds;
            public long Launches;
        }

        [StructLayout(LayoutKind.Sequential)]
        public struct Scan
        {
            public long Tokens;
            public int Sequences, Dim, State, Groups, DeltaSoftplus;
            public IntPtr Offsets;
            public IntPtr U, Delta, Z, A, B, C, D, DeltaBias, H0;
            public long LdU, LdDelta, LdZ, LdB, LdC;
        }

        [StructLayout(LayoutKind.Sequential)]
        public struct ScanGradients
        {
            public IntPtr Du, Ddelta, Dz, DA, DB, DC, DD, DdeltaBias, Dh0;
            public long LdDu, LdDdelta, LdDz, LdDB, LdDC;
        }

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_init(int device, out IntPtr out_ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_shutdown(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern IntPtr prad_last_error();

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern IntPtr prad_version();

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_set_option(IntPtr ctx, [MarshalAs(UnmanagedType.LPStr)] string key, [MarshalAs(UnmanagedType.LPStr)] string value);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sync(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_launch_count(IntPtr ctx, out long out_count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_stream(IntPtr ctx, out IntPtr out_stream);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_use_stream(IntPtr ctx, IntPtr stream);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_device_info(IntPtr ctx, out DeviceInfo @out);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_measure_pipe_rate(IntPtr ctx, int pipe, out double out_tflops);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_selftest_bounded_wait(IntPtr ctx, int polls);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_timing_begin(IntPtr ctx, [MarshalAs(UnmanagedType.LPStr)] string label);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_timing_end(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_get_timings(IntPtr ctx, [In, Out] Timing[] @out, int capacity, out int out_count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_alloc(IntPtr ctx, UIntPtr bytes, out IntPtr out_dptr);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_free(IntPtr ctx, IntPtr dptr);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_zero(IntPtr ctx, IntPtr dptr, UIntPtr bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_copy(IntPtr ctx, IntPtr dst, IntPtr src, UIntPtr bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_copy_2d(IntPtr ctx, IntPtr dst, UIntPtr dst_pitch, IntPtr src, UIntPtr src_pitch, UIntPtr width_bytes, UIntPtr rows);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload(IntPtr ctx, IntPtr dst, IntPtr src_host, UIntPtr bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_download(IntPtr ctx, IntPtr dst_host, IntPtr src, UIntPtr bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload_prefetch(IntPtr ctx, IntPtr dst, IntPtr src_host, UIntPtr bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload_join(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload_fence(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload_rows(IntPtr ctx, IntPtr dst, IntPtr[] src_rows, int rows, UIntPtr row_bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_download_rows(IntPtr ctx, IntPtr[] dst_rows, IntPtr src, int rows, UIntPtr row_bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_download_many(IntPtr ctx, IntPtr dst_host, IntPtr[] srcs_host, UIntPtr[] bytes_host, int count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_upload_many(IntPtr ctx, IntPtr[] dsts_host, IntPtr src_host, UIntPtr[] bytes_host, int count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_slot_store(IntPtr ctx, IntPtr guid_16_bytes, IntPtr[] ptrs_host, UIntPtr[] bytes_host, int count, int copy);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_slot_restore(IntPtr ctx, IntPtr guid_16_bytes, [Out] IntPtr[] out_ptrs_host, int count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_slot_drop(IntPtr ctx, IntPtr guid_16_bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_slot_count(IntPtr ctx, out int out_count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_alloc_host(IntPtr ctx, UIntPtr bytes, out IntPtr out_hptr);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_free_host(IntPtr ctx, IntPtr hptr);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_gemm(IntPtr ctx, DType dt, int transA, int transB, int M, int N, int K, double alpha, IntPtr A, int lda, IntPtr B, int ldb, double beta, IntPtr C, int ldc, int batch, long strideA, long strideB, long strideC);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_packed_create(IntPtr ctx, int rows, int cols, int forms, int block_rows_form, int block_cols_form, IntPtr @out);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_packed_destroy(IntPtr p);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_packed_shape(IntPtr p, IntPtr rows, IntPtr cols, IntPtr forms, IntPtr block_rows_form, IntPtr block_cols_form);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_pack(IntPtr p, IntPtr x, long ld);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_act_forward_pack(IntPtr p, Act act, IntPtr x, IntPtr y, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_act_backward_pack(IntPtr p, Act act, IntPtr saved, IntPtr dy, IntPtr dx, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_mse_act_backward_pack(IntPtr p, Act act, IntPtr saved, IntPtr output, IntPtr target, long rows_total, IntPtr dx, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_packed_column_sums(IntPtr p, IntPtr @out);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_layernorm_pack(IntPtr p, IntPtr x, IntPtr residual, IntPtr sum, IntPtr mean, IntPtr stdv);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_layernorm_backward_pack(IntPtr p, IntPtr x, IntPtr mean, IntPtr stdv, IntPtr dy, IntPtr residual, IntPtr dx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_gemm_packed(IntPtr ctx, IntPtr A, int form_a, IntPtr B, int form_b, double alpha, double beta, IntPtr C, long ldc, IntPtr bias);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_forward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr Y, int M, int K, int N, IntPtr bias, IntPtr Z_out, Act act, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_backward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr dC, IntPtr dA, IntPtr dB, int M, int K, int N, int accumulate_dB, double dB_scale, Act act_below, IntPtr saved_below, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_act_backward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr dOut, Act act, IntPtr saved, double act_alpha, IntPtr dPre, IntPtr dA, IntPtr dB, int M, int K, int N);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_act_backward_host(IntPtr ctx, DType dt, IntPtr A_host, IntPtr B_host, IntPtr dOut_host, Act act, IntPtr saved_host, double act_alpha, IntPtr dPre_host, IntPtr dA_host, IntPtr dB_host, int M, int K, int N);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_batch_matmul_forward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr C, int depth, int M, int K, int N, int b_shared);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_batch_matmul_backward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr dC, IntPtr dA, IntPtr dB, IntPtr dB_mean, int depth, int M, int K, int N, int b_shared);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_window_attention_forward(IntPtr ctx, DType dt, IntPtr qkv, IntPtr P, IntPtr @out, int windows, int window, int heads, int head_dim, double scale);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_window_attention_backward(IntPtr ctx, DType dt, IntPtr qkv, IntPtr P, IntPtr d_out, IntPtr d_qkv, int windows, int window, int heads, int head_dim, double scale);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_and_sum_forward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr @out, int R, int C, int N, int P);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_matmul_and_sum_backward(IntPtr ctx, DType dt, IntPtr A, IntPtr B, IntPtr dOut, IntPtr dA, IntPtr dB, int R, int C, int N, int P);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_act_forward(IntPtr ctx, DType dt, Act act, IntPtr x, IntPtr y, long n, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_act_backward(IntPtr ctx, DType dt, Act act, IntPtr saved, IntPtr dy, IntPtr dx, long n, double act_alpha);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_swish_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr beta, IntPtr y, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_swish_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr beta, IntPtr dy, IntPtr dx, IntPtr dbeta, long n, int accumulate);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_swiglu_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr w, IntPtr v, IntPtr b, IntPtr c, double beta, IntPtr y, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_swiglu_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr w, IntPtr v, IntPtr b, IntPtr c, double beta, IntPtr dy, IntPtr dx, IntPtr dw, IntPtr dv, IntPtr db, IntPtr dc, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_hadamard_forward(IntPtr ctx, DType dt, IntPtr a, IntPtr b, IntPtr y, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_hadamard_backward(IntPtr ctx, DType dt, IntPtr a, IntPtr b, IntPtr dy, IntPtr da, IntPtr db, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_lstm_cell_backward(IntPtr ctx, DType dt, long n, IntPtr h, IntPtr target, double loss_scale, IntPtr[] dh_contrib_host, int n_contrib, IntPtr dc_next, IntPtr[] gates_ifgo_host, IntPtr tanh_c, IntPtr c_prev, IntPtr[] dpre_ifgo_host, IntPtr dc_prev);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_lstm_forward(IntPtr ctx, DType dt, int steps, int batch, int hidden, IntPtr U, IntPtr[] bias_ifgo_host, IntPtr pre, IntPtr[] gates_ifgo_host, IntPtr C, IntPtr tanh_c, IntPtr H, IntPtr H_prev, IntPtr FC, IntPtr IG);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_lstm_backward(IntPtr ctx, DType dt, int steps, int batch, int hidden, IntPtr U, IntPtr H, IntPtr target, double loss_scale, IntPtr[] gates_ifgo_host, IntPtr tanh_c, IntPtr C, IntPtr dpre, IntPtr scratch);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_add_forward(IntPtr ctx, DType dt, IntPtr a, IntPtr b, IntPtr c, IntPtr y, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_add_broadcast_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr bias, IntPtr y, int rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_add_broadcast_backward(IntPtr ctx, DType dt, IntPtr dy, IntPtr dbias, int rows, int cols, int accumulate);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_column_sums(IntPtr ctx, DType dt, IntPtr x, int rows, int cols, int batch, long stride, double scale, IntPtr @out, long out_stride);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_add_broadcast_backward_static(IntPtr stream, DType dt, IntPtr dy, IntPtr dbias, int rows, int cols, int accumulate);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_scale(IntPtr ctx, DType dt, IntPtr x, IntPtr y, long n, double s);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_transpose(IntPtr ctx, DType dt, IntPtr x, IntPtr y, int rows, int cols, int depth);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_softmax_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr y, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_softmax_backward(IntPtr ctx, DType dt, IntPtr y, IntPtr dy, IntPtr dx, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sine_softmax_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr y, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sine_softmax_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr dy, IntPtr dx, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_layernorm_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr y, IntPtr mean, IntPtr stdv, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_layernorm_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr mean, IntPtr stdv, IntPtr dy, IntPtr dx, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_layernorm_backward_add(IntPtr ctx, DType dt, IntPtr x, IntPtr mean, IntPtr stdv, IntPtr dy, IntPtr residual, IntPtr dx, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_row_sum_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr y, long rows, int cols, int average);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_row_sum_backward(IntPtr ctx, DType dt, IntPtr dy, IntPtr dx, long rows, int cols, int average);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_broadcast_forward(IntPtr ctx, DType dt, IntPtr x, int in_rows, int in_cols, IntPtr y, int out_rows, int out_cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_broadcast_backward(IntPtr ctx, DType dt, IntPtr dy, int out_rows, int out_cols, IntPtr dx, int in_rows, int in_cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_batchnorm_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr y, IntPtr stats, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_batchnorm_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr stats, IntPtr dy, IntPtr dx, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_scale_shift_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr beta, IntPtr gamma, IntPtr y, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_scale_shift_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr beta, IntPtr dy, IntPtr dx, IntPtr dbeta, IntPtr dgamma, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_rmsnorm_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr g, IntPtr y, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_rmsnorm_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr g, IntPtr dy, IntPtr dx, IntPtr dg, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_group_norm_forward(IntPtr ctx, DType dt, IntPtr x, IntPtr gamma, IntPtr beta, IntPtr y, IntPtr mean, IntPtr rstd, long samples, long positions, int channels, int groups, double eps, int swish);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_group_norm_backward(IntPtr ctx, DType dt, IntPtr x, IntPtr gamma, IntPtr beta, IntPtr mean, IntPtr rstd, IntPtr dy, IntPtr dx, IntPtr dgamma, IntPtr dbeta, long samples, long positions, int channels, int groups, int swish);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dropout(IntPtr ctx, DType dt, IntPtr x, IntPtr residual, IntPtr y, long n, double p, ulong seed, ulong offset, IntPtr step);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_causal_conv_forward(IntPtr ctx, DType dt, IntPtr x, long ld_x, IntPtr w, IntPtr bias, IntPtr state, IntPtr offsets, IntPtr y, long ld_y, IntPtr state_out, int sequences, long tokens, int dim, int width, int swish);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_causal_conv_backward(IntPtr ctx, DType dt, IntPtr x, long ld_x, IntPtr w, IntPtr bias, IntPtr state, IntPtr offsets, IntPtr dy, long ld_dy, IntPtr dx, long ld_dx, IntPtr dw, IntPtr dbias, IntPtr dstate, int sequences, long tokens, int dim, int width, int swish);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_causal_conv_step(IntPtr ctx, DType dt, IntPtr x, long ld_x, IntPtr w, IntPtr bias, IntPtr state, IntPtr y, long ld_y, IntPtr state_out, long batch, int dim, int width, int swish);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_selective_scan_saved_bytes(DType dt, ref Scan scan, out UIntPtr out_bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_selective_scan_forward(IntPtr ctx, DType dt, ref Scan scan, IntPtr y, long ld_y, IntPtr h_last, IntPtr saved);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_selective_scan_backward(IntPtr ctx, DType dt, ref Scan scan, IntPtr saved, IntPtr dy, long ld_dy, ref ScanGradients gradients);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_selective_scan_step(IntPtr ctx, DType dt, ref Scan scan, IntPtr y, long ld_y, IntPtr h_out);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_mse_forward(IntPtr ctx, DType dt, IntPtr @out, IntPtr target, IntPtr loss_out, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_mse_backward(IntPtr ctx, DType dt, IntPtr @out, IntPtr target, IntPtr grad, long rows, int cols, long rows_total);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_cce_forward(IntPtr ctx, DType dt, IntPtr @out, IntPtr target, IntPtr loss_out, long rows, int cols);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_cce_backward(IntPtr ctx, DType dt, IntPtr @out, IntPtr target, IntPtr grad, long rows, int cols, long rows_total);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_embedding_forward(IntPtr ctx, DType dt, IntPtr index_col, IntPtr W, IntPtr @out, int n, int vocab, int dim);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_embedding_backward(IntPtr ctx, DType dt, IntPtr index_col, IntPtr dOut, IntPtr dW, int n, int vocab, int dim);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_segmented_sum(IntPtr ctx, DType dt, IntPtr[] srcs_host, int count, IntPtr @out, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_accumulate(IntPtr ctx, DType dt, IntPtr dest, IntPtr src, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_batch_mean(IntPtr ctx, DType dt, IntPtr[] srcs_host, int count, IntPtr @out, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_clip_reference(IntPtr ctx, DType dt, IntPtr[] grads_host, long[] sizes_host, int count, double clip_value, double min_value);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_clip_global_norm(IntPtr ctx, DType dt, IntPtr[] grads_host, long[] sizes_host, int count, double max_norm, IntPtr norm_out);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_adam(IntPtr ctx, DType dt, IntPtr[] w_host, IntPtr[] g_host, IntPtr[] m_host, IntPtr[] v_host, long[] sizes_host, int count, double lr, double beta1, double beta2, double eps, double iteration, AdamForm form, int zero_grad);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_clip_adam(IntPtr ctx, DType dt, IntPtr[] w_host, IntPtr[] g_host, IntPtr[] m_host, IntPtr[] v_host, long[] sizes_host, int count, int clip_mode, double clip_value, double min_value, double lr, double beta1, double beta2, double eps, double iteration, AdamForm form, int zero_grad);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_create(IntPtr ctx, DType dt, out IntPtr out_graph);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_destroy(IntPtr g);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_add_value(IntPtr g, int rows, int cols, IntPtr data, out int out_value);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_add_deep_value(IntPtr g, int depth, int rows, int cols, IntPtr data, out int out_value);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_set_gradient_destination(IntPtr g, int value, IntPtr grad_matrix);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_set_result_copy(IntPtr g, int value, IntPtr matrix);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_add_node(IntPtr g, Op op, int[] in_values, int n_in, int out_value, double scalar, out int out_node);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_forward(IntPtr g);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_backward(IntPtr g, int start_value, IntPtr d_start);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_backward_multi(IntPtr g, int[] start_values, IntPtr[] d_starts, int count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_value_data(IntPtr g, int value, out IntPtr out_data);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_value_gradient(IntPtr g, int value, out IntPtr out_grad);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_consumer_count(IntPtr g, int value, out int out_count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_graph_plan_products(IntPtr g, out long out_forward, out long out_backward);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_unary(IntPtr ctx, DType dt, TensorOp op, IntPtr x, IntPtr y, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_unary_reverse(IntPtr ctx, DType dt, TensorOp op, IntPtr saved, IntPtr dy, IntPtr dx, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_binary(IntPtr ctx, DType dt, TensorOp op, IntPtr a, IntPtr b, IntPtr y, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_binary_reverse(IntPtr ctx, DType dt, TensorOp op, IntPtr a, IntPtr b, IntPtr dy, IntPtr da, IntPtr db, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_matmul(IntPtr ctx, DType dt, IntPtr A, int a_rows, int a_cols, IntPtr B, int b_rows, int b_cols, double alpha, double beta, IntPtr C);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_matmul_reverse(IntPtr ctx, DType dt, IntPtr A, int a_rows, int a_cols, IntPtr B, int b_rows, int b_cols, IntPtr dC, IntPtr dA, IntPtr dB);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_gather(IntPtr ctx, DType dt, IntPtr x, long outer, int axis_len, long inner, IntPtr indices, int count, IntPtr y);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_gather_reverse(IntPtr ctx, DType dt, IntPtr upstream, long outer, int axis_len, long inner, IntPtr indices, int count, IntPtr dx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_tile(IntPtr ctx, DType dt, IntPtr x, int rows, int cols, int mult_rows, int mult_cols, IntPtr y);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_tensor_tile_reverse(IntPtr ctx, DType dt, IntPtr upstream, int rows, int cols, int mult_rows, int mult_cols, IntPtr dx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_capture_begin(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_capture_end(IntPtr ctx, out IntPtr out_sequence);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sequence_launch(IntPtr ctx, IntPtr sequence);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sequence_launch_count(IntPtr sequence, out long out_count);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_sequence_destroy(IntPtr ctx, IntPtr sequence);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_unique_id(IntPtr out_id_128_bytes);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_init(IntPtr ctx, IntPtr id_128_bytes, int rank, int world_size);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_allreduce(IntPtr ctx, DType dt, IntPtr buf, long n);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_wait(IntPtr ctx);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_reduce(IntPtr ctx, DType dt, IntPtr buf, long n, int root);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_broadcast(IntPtr ctx, DType dt, IntPtr buf, long n, int root);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_mark(IntPtr ctx, int slot);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_wait_mark(IntPtr ctx, int slot);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_wait_host(IntPtr ctx, double timeout_ms);

        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]
        public static extern int prad_dp_shutdown(IntPtr ctx);

        /// <summary>Maps a status to the exception the managed operation would have thrown.</summary>
        public static void Check(int status)
        {
            if (status == 0)
            {
                return;
            }

            string msg = Marshal.PtrToStringAnsi(prad_last_error()) ?? "libprad_cuda error";
            switch ((Status)status)
            {
                case Status.ErrShape: throw new InvalidOperationException(msg);           // MatrixMultiplyOperation.cs:59-62
                case Status.ErrNotInitialized: throw new CudaNotInitializedException();    // GpuMatrixMultiplyOperation.cs:115-118
                case Status.ErrInvalid: throw new ArgumentException(msg);
                case Status.ErrOom: throw new OutOfMemoryException(msg);
                case Status.ErrTimeout: throw new TimeoutException(msg);                   // visitor TimeoutInMinutes
                default: throw new InvalidOperationException("CUDA failure: " + msg);     // CudaBlas.cs:251-256
            }
        }
    }

    /// <summary>A dense row-major matrix (or DeepMatrix: depth consecutive matrices) resident on the device.</summary>
    public sealed class DeviceMatrix : IDisposable
    {
        public DeviceMatrix(IntPtr ctx, PradCuda.DType dtype, int rows, int cols, int depth = 1)
        {
            this.Ctx = ctx;
            this.DType = dtype;
            this.Rows = rows;
            this.Cols = cols;
            this.Depth = depth;
            PradCuda.Check(PradCuda.prad_alloc(ctx, (UIntPtr)this.Bytes, out IntPtr p));
            this.Ptr = p;
        }

        public IntPtr Ctx { get; }

        public IntPtr Ptr { get; private set; }

        public PradCuda.DType DType { get; }

        public int Rows { get; }

        public int Cols { get; }

        public int Depth { get; }

        public int ElementSize => this.DType == PradCuda.DType.F64 ? 8 : 4;

        public ulong Bytes => (ulong)this.Rows * (ulong)this.Cols * (ulong)this.Depth * (ulong)this.ElementSize;

        /// <summary>Uploads a jagged double[][] / float[][] (pinned row by row) with one call.</summary>
        public void Upload(Array[] rows)
        {
            var handles = new GCHandle[rows.Length];
            var ptrs = new IntPtr[rows.Length];
            try
            {
                for (int i = 0; i < rows.Length; ++i)
                {
                    handles[i] = GCHandle.Alloc(rows[i], GCHandleType.Pinned);
                    ptrs[i] = handles[i].AddrOfPinnedObject();
                }

                PradCuda.Check(PradCuda.prad_upload_rows(this.Ctx, this.Ptr, ptrs, rows.Length, (UIntPtr)((ulong)this.Cols * (ulong)this.ElementSize)));
                PradCuda.Check(PradCuda.prad_sync(this.Ctx));
            }
            finally
            {
                foreach (var h in handles)
                {
                    if (h.IsAllocated)
                    {
                        h.Free();
                    }
                }
            }
        }

        /// <summary>Downloads into a jagged array of the same shape (blocks until the copy is done).</summary>
        public void Download(Array[] rows)
        {
            var handles = new GCHandle[rows.Length];
            var ptrs = new IntPtr[rows.Length];
            try
            {
                for (int i = 0; i < rows.Length; ++i)
                {
                    handles[i] = GCHandle.Alloc(rows[i], GCHandleType.Pinned);
                    ptrs[i] = handles[i].AddrOfPinnedObject();
                }

                PradCuda.Check(PradCuda.prad_download_rows(this.Ctx, ptrs, this.Ptr, rows.Length, (UIntPtr)((ulong)this.Cols * (ulong)this.ElementSize)));
            }
            finally
            {
                foreach (var h in handles)
                {
                    if (h.IsAllocated)
                    {
                        h.Free();
                    }
                }
            }
        }

        public void Dispose()
        {
            if (this.Ptr != IntPtr.Zero)
            {
                PradCuda.prad_free(this.Ctx, this.Ptr);
                this.Ptr = IntPtr.Zero;
            }
        }
    }
}
